// Attention of single tokens over a cache in pages: m40llm_attention_paged_async.
//
// Rows are split over their entries: softmax statistics are kept with a running maximum in base 2, and the parts' (maximum, sum, unnormalised output) meet in a fixed
// order: in clusters of CTAs for short rows, else in a join behind the kernel that made them. Where accumulated weights are asked for, the scores are kept in scratch
// and turned into weights once the maximum and sum of every row are known.
//   paged_tiles_kernel  f16 entries, head sizes 64 and 128: matrix instructions on 64-entry tiles
//   paged_lanes_kernel  (attention_paged_lanes.cu) f32 entries and other f16 head sizes, rows in 16-byte pieces: f32 multiply-adds in registers
//   paged_rows_kernel   what is left, odd head sizes and alignments: f32 multiply-adds on tiles in shared memory
#include "attention_paged.cuh"
#include "stack_math.cuh"
#include "tc_ptx.cuh"
#include <type_traits>

namespace {

using namespace attn_mma;

// The part of them that split s covers: whole tiles of 64, counted from the one that `begin` lies in, dealt evenly to the splits, at least a.chunk
// entries to each that has any.
__device__ __forceinline__ void paged_chunk(const PagedAttnArgs& a, uint32_t split, uint32_t begin, uint32_t end, uint32_t* t0, uint32_t* t1) {
    const uint32_t from = begin & ~63u, tiles = end > from ? (end - from + 63u) / 64u : 0u;
    const uint32_t chunk = max((tiles + a.splits - 1u) / a.splits * 64u, a.chunk);
    const uint64_t lo = (uint64_t)from + (uint64_t)split * chunk, hi = lo + chunk;
    *t0 = lo > begin ? (lo < end ? (uint32_t)lo : end) : begin;
    *t1 = hi < end ? (uint32_t)hi : end;
    if (*t1 < *t0) *t1 = *t0;
}

constexpr uint32_t ROWS_THREADS = 128;

// CTA = (row, GT q heads of one kv head, chunk). Tiles of T entries of keys and values in shared memory, two in flight. Scores: thread =
// (entry, slice of the dimensions), the slices meet in shared memory; softmax: warp = head, lane = entry; output: thread = dimensions.
template <typename ET, int GT, int DV>
__global__ void __launch_bounds__(ROWS_THREADS) paged_rows_kernel(PagedAttnArgs a, uint32_t T, uint32_t vec, uint32_t pitch) {
    extern __shared__ __align__(128) unsigned char smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, hd = a.c.hd, hd4 = (hd + 3u) & ~3u;
    float* s_q = reinterpret_cast<float*>(smem);                 // [GT][hd4]
    float* s_part = s_q + GT * hd4;                              // [slices][GT][T]
    float* s_p = s_part + ROWS_THREADS * GT;                     // [GT][32]
    float* s_corr = s_p + GT * 32;                               // [GT]
    uint32_t* s_ok = reinterpret_cast<uint32_t*>(s_corr + 8);    // [2][32]
    ET* s_k = reinterpret_cast<ET*>(s_ok + 64);                  // [2][T][pitch]
    ET* s_v = s_k + 2u * T * pitch;
    pdl_wait();
    pdl_trigger();
    const uint32_t split = blockIdx.x, row = blockIdx.z, subgroups = (a.group + GT - 1) / GT;
    const uint32_t kvh = blockIdx.y / subgroups, g0 = (blockIdx.y % subgroups) * GT, G = min((uint32_t)GT, a.group - g0);
    const uint32_t head0 = kvh * a.group + g0;
    uint32_t slot, begin, end, t0 = 0, t1 = 0;
    const bool inside = paged_row_range(a, row, &slot, &begin, &end);
    if (!inside && tid == 0 && split == 0 && blockIdx.y == 0) atomicOr(a.status, 1u);
    if (inside) paged_chunk(a, split, begin, end, &t0, &t1);
    const bool partial = a.splits > 1 || a.scores;
    float acc[GT][DV];
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
        for (int j = 0; j < DV; ++j) acc[g][j] = 0.0f;
    float m_run[(GT + 3) / 4], l_run[(GT + 3) / 4];  // heads warp, warp + 4, ..
#pragma unroll
    for (int j = 0; j < (GT + 3) / 4; ++j) m_run[j] = -INFINITY, l_run[j] = 0.0f;

    for (uint32_t i = tid; i < GT * hd4; i += ROWS_THREADS) {
        const uint32_t g = i / hd4, d = i % hd4;
        s_q[i] = g < G && d < hd ? a.q[((size_t)row * a.q_heads + head0 + g) * hd + d] * a.scale : 0.0f;
    }
    const uint32_t tiles = (t1 - t0 + T - 1) / T;
    const ET* K = reinterpret_cast<const ET*>(a.c.k);
    const ET* V = reinterpret_cast<const ET*>(a.c.v);
    // entries past the end and on pages outside the pool read as zeros and are masked
    auto load = [&](uint32_t tile) {
        const uint32_t base = t0 + tile * T, buf = tile & 1u;
        ET* dk = s_k + (size_t)buf * T * pitch;
        ET* dv = s_v + (size_t)buf * T * pitch;
        constexpr uint32_t VE = 16u / sizeof(ET);
        const uint32_t pieces = vec ? hd / VE : hd4;
        for (uint32_t i = tid; i < T * pieces; i += ROWS_THREADS) {
            const uint32_t r = i / pieces, p = i % pieces, e = base + r;
            const uint32_t page = e < t1 ? paged_page(a.c, slot, e) : PAGED_NONE;
            const bool ok = page != PAGED_NONE;
            const size_t src = ok ? paged_row(a.c, page, kvh, e) : 0;
            if (p == 0) {
                s_ok[buf * 32u + r] = ok;
                if (e < t1 && !ok) atomicOr(a.status, 1u);
            }
            if (vec) {
                if (ok) {
                    cp_async16(dk + r * pitch + p * VE, K + src + p * VE);
                    cp_async16(dv + r * pitch + p * VE, V + src + p * VE);
                } else {
                    *reinterpret_cast<uint4*>(dk + r * pitch + p * VE) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(dv + r * pitch + p * VE) = make_uint4(0, 0, 0, 0);
                }
            } else {
                const bool in = ok && p < hd;
                dk[r * pitch + p] = in ? K[src + p] : ET(0.0f);
                dv[r * pitch + p] = in ? V[src + p] : ET(0.0f);
            }
        }
    };
    if (tiles) load(0);
    cp_async_commit();
    const uint32_t slices = ROWS_THREADS / T, my = tid % T, slice = tid / T;
    for (uint32_t tile = 0; tile < tiles; ++tile) {
        if (tile + 1 < tiles) load(tile + 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        const uint32_t buf = tile & 1u, base = t0 + tile * T;
        {
            const ET* kr = s_k + ((size_t)buf * T + my) * pitch;
            float s[GT];
#pragma unroll
            for (int g = 0; g < GT; ++g) s[g] = 0.0f;
            for (uint32_t d = slice * 4u; d < hd4; d += slices * 4u) {
                const float k0 = m40_load_elem(kr + d), k1 = m40_load_elem(kr + d + 1), k2 = m40_load_elem(kr + d + 2), k3 = m40_load_elem(kr + d + 3);
#pragma unroll
                for (int g = 0; g < GT; ++g) {
                    const float4 x = *reinterpret_cast<const float4*>(s_q + g * hd4 + d);
                    s[g] = fmaf(x.x, k0, fmaf(x.y, k1, fmaf(x.z, k2, fmaf(x.w, k3, s[g]))));
                }
            }
#pragma unroll
            for (int g = 0; g < GT; ++g) s_part[(slice * GT + g) * T + my] = s[g];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < (GT + 3) / 4; ++j) {
            const uint32_t g = warp + 4u * j;
            if (g >= (uint32_t)GT) break;
            float s = -INFINITY;
            const uint32_t e = base + lane;
            if (lane < T && s_ok[buf * 32u + lane]) {
                s = 0.0f;
                for (uint32_t i = 0; i < slices; ++i) s += s_part[(i * GT + g) * T + lane];
            }
            if (a.scores && g < G && lane < T && e < t1) a.scores[((size_t)row * a.q_heads + head0 + g) * a.ld_scores + e] = s;
            const float m_new = fmaxf(m_run[j], warp_max(s)), m_use = m_new == -INFINITY ? 0.0f : m_new;
            const float corr = exp2f(m_run[j] - m_use), p = exp2f(s - m_use);
            l_run[j] = l_run[j] * corr + warp_sum(p);
            m_run[j] = m_new;
            s_p[g * 32u + lane] = p;
            if (lane == 0) s_corr[g] = corr;
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            const float c = s_corr[g];
#pragma unroll
            for (int j = 0; j < DV; ++j) acc[g][j] *= c;
        }
        const ET* vt = s_v + (size_t)buf * T * pitch;
        for (uint32_t t = 0; t < T; t += 4) {
            float v[4][DV];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < DV; ++j) {
                    const uint32_t d = tid + ROWS_THREADS * j;
                    v[u][j] = d < hd ? m40_load_elem(vt + (t + u) * pitch + d) : 0.0f;
                }
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const float4 p = *reinterpret_cast<const float4*>(s_p + g * 32u + t);
#pragma unroll
                for (int j = 0; j < DV; ++j) acc[g][j] = fmaf(p.x, v[0][j], fmaf(p.y, v[1][j], fmaf(p.z, v[2][j], fmaf(p.w, v[3][j], acc[g][j]))));
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();
#pragma unroll
    for (int j = 0; j < (GT + 3) / 4; ++j) {
        const uint32_t g = warp + 4u * j;
        if (g < G && lane == 0) {
            if (partial) {
                const size_t pi = ((size_t)row * a.q_heads + head0 + g) * a.splits + split;
                a.part_m[pi] = m_run[j];
                a.part_l[pi] = l_run[j];
            }
            s_corr[g] = l_run[j];
        }
    }
    __syncthreads();
    if (partial && t1 <= t0) return;  // an empty part: l = 0, its outputs are not read
#pragma unroll
    for (int g = 0; g < GT; ++g)
        if ((uint32_t)g < G) {
            const size_t head = (size_t)row * a.q_heads + head0 + g;
            const float l = s_corr[g], inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
            for (int j = 0; j < DV; ++j) {
                const uint32_t d = tid + ROWS_THREADS * j;
                if (d >= hd) continue;
                if (partial)
                    a.part_o[(head * a.splits + split) * hd + d] = acc[g][j];
                else
                    a.out[head * hd + d] = l > 0.0f || isnan(l) ? acc[g][j] * (isnan(l) ? l : inv) : 0.0f;
            }
        }
}

constexpr uint32_t TILE = 16, TILES_THREADS = 128, TILES_WARPS = TILES_THREADS / 32, SPAN = TILE * TILES_WARPS;

// One q head over the entries [t0, t1) of one kv head by one warp in plain f32: what the matrix instructions cannot give where keys or values are not finite (a part of 0, or of the other sign, times an infinity is NaN). Lane = dimensions
// 2 lane, 2 lane + 1 (+ 64). Results as in paged_tiles_kernel.
template <int HD>
__device__ __noinline__ void paged_plain_run(const PagedAttnArgs& a, uint32_t slot, uint32_t kvh, const float* q, float* scores, uint32_t t0,
                                             uint32_t t1, uint32_t share, float bias, float* m_out, float* l_out, float* o_out) {
    const uint32_t lane = threadIdx.x & 31u, d = 2u * lane;
    const __half* K = reinterpret_cast<const __half*>(a.c.k);
    const __half* V = reinterpret_cast<const __half*>(a.c.v);
    float x[HD / 32], o[HD / 32], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) {
        x[2 * j] = q[d + 64 * j] * a.scale, x[2 * j + 1] = q[d + 64 * j + 1] * a.scale;
        o[2 * j] = o[2 * j + 1] = 0.0f;
    }
    for (uint32_t e = t0; e < t1; ++e) {
        if (e / TILE % TILES_WARPS != share) continue;
        const uint32_t page = paged_page(a.c, slot, e);
        if (page == PAGED_NONE) continue;
        const size_t at = paged_row(a.c, page, kvh, e) + d;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
            const float2 k = __half22float2(*reinterpret_cast<const __half2*>(K + at + 64 * j));
            s += x[2 * j] * k.x + x[2 * j + 1] * k.y;
        }
        s = warp_sum(s);
        if (scores && lane == 0) scores[e] = s;
        const float m_new = fmaxf(m, s - bias), use = m_new == -INFINITY ? 0.0f : m_new;
        const float corr = m == -INFINITY ? 0.0f : exp2f(m - m_new), p = exp2f(s - use);
        l = l * corr + p;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(V + at + 64 * j));
            o[2 * j] = o[2 * j] * corr + p * v.x, o[2 * j + 1] = o[2 * j + 1] * corr + p * v.y;
        }
        m = m_new;
    }
    if (lane == 0) *m_out = m, *l_out = l;
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) *reinterpret_cast<float2*>(o_out + d + 64 * j) = make_float2(o[2 * j], o[2 * j + 1]);
}

__device__ __forceinline__ void ldmatrix_at(uint32_t (&r)[4], uint32_t smem) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem) : "memory");
}
__device__ __forceinline__ void ldmatrix_trans_at(uint32_t (&r)[4], uint32_t smem) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem) : "memory");
}

// Weights are relative to the maximum less 15: f16 then holds a small one down to 2^-40 of the largest instead of 2^-25. That reference, as it is
// rounded, is what a part carries as its maximum.
constexpr float WEIGHT_BIAS = 15.0f;

// Without a list: the place of a CTA that takes unit `unit` of row `row` from its first tile on, in a list of that row alone. False for a row without entries, whose zeros
// are written. All threads of the CTA.
template <int HD>
__device__ __forceinline__ bool paged_direct_enter(const PagedAttnArgs& a, PagedList& s, uint32_t row, uint32_t unit, PagedPlace& p) {
    uint32_t slot, begin, end;
    const bool inside = paged_row_range(a, row, &slot, &begin, &end);
    if (!inside || end <= begin) {
        const uint32_t subgroups = (a.group + a.heads_at_once - 1u) / a.heads_at_once, kvh = unit / subgroups;
        const uint32_t g0 = (unit - kvh * subgroups) * a.heads_at_once, G = min(a.heads_at_once, a.group - g0);
        float* out = a.out + ((size_t)row * a.q_heads + kvh * a.group + g0) * HD;
        for (uint32_t i = threadIdx.x; i < G * HD; i += TILES_THREADS) out[i] = 0.0f;
        if (!inside && unit == 0 && threadIdx.x == 0) atomicOr(a.status, 1u);
        return false;
    }
    if (threadIdx.x == 0) s.slot[0] = slot, s.begin[0] = begin, s.end[0] = end;
    __syncthreads();
    p.row = 0, p.unit = unit, p.tile = 0;
    paged_list_enter(s, p, SPAN);
    return true;
}

constexpr uint32_t DIRECT_CLUSTER = 8;

// A run of the list of work per CTA, tiles of 64 entries; a warp takes 16 of them, with a ring of its own. Against one CTA per (row, unit, 1024
// entries): 32 rows of up to 16384 entries 198 -> 173 us (179 to 181 on other B200s), one of 130001 110 -> 90. Runs of single warps spread the reads over four times as many places,
// and without a barrier per tile the warps drift apart: 187 and 179 us for the 32 rows.
//   ring      K and V tiles by cp.async, looked up in the page table as they are fetched, XOR-swizzled; it runs on across units.
//   S = Q K^T, O += P V   mma.sync m16n8k16 with f32 sums. Queries and weights are cut into f16 hi + lo, which leaves 2^-22 of them; a head's query is
//                         brought to 2^9 .. 2^10 by a power of two first (its largest value), as the lo of a small value would lose its bits. A group has
//                         at most 8 heads as a rule: hi and lo are then the two halves of the 16 rows of ONE operand, and the halves of the result are
//                         added (WIDE: two products).
//   softmax               online in base 2; the outputs are rescaled only when a maximum moved.
template <int HD, bool WIDE>
struct TilesCfg {
    static constexpr int STAGES = HD == 128 ? 3 : 4, CTAS = HD == 128 ? 2 : 3;
    static constexpr int STAGE = 2 * (int)TILE * HD * 2;                                                                    // K and V of a tile
    static constexpr int SMEM = 256 + (int)TILES_WARPS * STAGES * STAGE + (int)sizeof(PagedList);  // rings, the list
    // DIRECT: what the CTAs of a cluster tell each other, by the teller's number: maxima and sums of the heads, outputs of the reader's share of the dimensions
    static constexpr int HEADS = WIDE ? 16 : 8, TOLD = (2 * (int)DIRECT_CLUSTER * HEADS + HEADS * HD) * 4;
};

// DIRECT, for short rows: a CTA per (row, unit), or a cluster of them with an equal share of the tiles each, puts its warps' parts together over the rings and writes the
// result, without a list and a join. In a cluster the CTAs store their parts into the memory of the one that puts the dimensions together.
template <int HD, bool WIDE, bool DIRECT>
__global__ void __launch_bounds__(TILES_THREADS, (TilesCfg<HD, WIDE>::CTAS)) paged_tiles_kernel(PagedAttnArgs a) {
    using Cfg = TilesCfg<HD, WIDE>;
    constexpr int KS = HD / 16, NT = HD / 8, CHUNKS = HD / 8, STAGES = Cfg::STAGES, ROWS = WIDE ? 16 : 8;
    static_assert(ROWS * (HD + 2) * 4 <= STAGES * Cfg::STAGE, "a warp's part lies over its ring");
    extern __shared__ __align__(128) unsigned char smem[];
    PagedList& list = *reinterpret_cast<PagedList*>(smem + 256 + TILES_WARPS * STAGES * Cfg::STAGE);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t4 = lane & 3u;
    const uint32_t units = a.c.kv_heads * ((a.group + a.heads_at_once - 1u) / a.heads_at_once), rows = DIRECT ? 1u : min(a.rows - a.row0, LIST_ROWS);
    pdl_wait();
    pdl_trigger();
    uint32_t peers = 1;
    if constexpr (DIRECT) asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(peers));
    const uint32_t worker = DIRECT ? blockIdx.x / peers : blockIdx.x, row0 = DIRECT ? worker / units : a.row0;
    PagedPlace at;
    uint32_t count;
    if constexpr (DIRECT) {
        if (!paged_direct_enter<HD>(a, list, row0, worker - row0 * units, at)) return;  // the same in every CTA of a cluster
        if (peers > 1u) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // it is there before anything is stored into it
        const uint32_t per = (at.tiles + peers - 1u) / peers;
        at.tile = min(tc::cluster_rank() * per, at.tiles);
        count = min(per, at.tiles - at.tile);
    } else {
        if (tid < 32u) paged_list_make(a, list, rows, SPAN);
        __syncthreads();
        const uint64_t total = list.prefix[rows] * units;
        const uint32_t workers = ctas_at_work(total, a.workers);
        if (worker >= workers) return;
        const uint64_t lo = quotient(worker * total, workers);
        count = (uint32_t)(quotient((worker + 1u) * total, workers) - lo);  // at least 1
        at = paged_list_at(list, lo, rows, units, SPAN);
    }

    // The lane copies piece `ch` of rows my_row, my_row + ROWS_AT_ONCE, ..; the swizzle of row r is r mod 8.
    constexpr uint32_t ROWS_AT_ONCE = 32u / CHUNKS, COPIES = TILE / ROWS_AT_ONCE, toSV = TILE * HD * 2u;
    const uint32_t ring = (((uint32_t)__cvta_generic_to_shared(smem) + 255u) & ~255u) + warp * (STAGES * Cfg::STAGE);  // whole rows, for the exclusive or below
    // DIRECT: outputs [ROWS][HD], maxima and sums of warp w
    const auto warp_part = [&](uint32_t w) { return reinterpret_cast<float*>(smem + w * (STAGES * Cfg::STAGE)); };
    const uint32_t subgroups = units / a.c.kv_heads;
    const uint32_t in_page = (1u << a.c.shift) - 1u, my_row = lane / CHUNKS, ch = lane % CHUNKS;
    const uint64_t head_bytes = (uint64_t)(HD * 2u) << a.c.shift;
    const uint64_t page_bytes = a.c.kv_heads * head_bytes;
    const ptrdiff_t toV = a.c.v - a.c.k;
    const uint32_t my_dst = ring + my_row * (HD * 2u) + ((ch ^ my_row) * 16u);  // my_row < 8; c * ROWS_AT_ONCE enters by exclusive or
    PagedPlace fetch = at;
    const uint32_t* pages = nullptr;
    const unsigned char* srcK = nullptr;
    bool bad = false;  // the warp met a page outside the pool
    auto aim = [&]() {
        pages = a.c.table + (size_t)list.slot[fetch.row] * a.c.max_pages;
        srcK = a.c.k + fetch.unit / subgroups * head_bytes + ch * 16u;
    };
    auto load = [&](uint32_t f) {  // tile f of the run, where `fetch` is
        const uint32_t base = fetch.first + fetch.tile * SPAN + warp * TILE, dst = my_dst + (f % STAGES) * Cfg::STAGE;
        if (a.c.shift >= 4u && base >= fetch.t0 && base + TILE <= fetch.t1) {  // a whole tile, within one page
            const uint32_t pg = pages[base >> a.c.shift];
            const bool ok = pg < a.c.pages;
            bad |= !ok;
            const unsigned char* src = srcK + (ok ? pg * page_bytes : 0) + ((base & in_page) + my_row) * (HD * 2u);
            const unsigned char* srcV = src + toV;
            const uint32_t bytes = ok ? 16u : 0u;
#pragma unroll
            for (uint32_t c = 0; c < COPIES; ++c) {
                const uint32_t to = (dst ^ ((c * ROWS_AT_ONCE & 7u) * 16u)) + c * (ROWS_AT_ONCE * HD * 2u);
                cp_async16_or_zero(to, src + c * (ROWS_AT_ONCE * HD * 2u), bytes);
                cp_async16_or_zero(to + toSV, srcV + c * (ROWS_AT_ONCE * HD * 2u), bytes);
            }
        } else if (base < fetch.t1 && base + TILE > fetch.t0) {
#pragma unroll 1
            for (uint32_t c = 0; c < COPIES; ++c) {
                const uint32_t e = base + c * ROWS_AT_ONCE + my_row;
                const bool in = e >= fetch.t0 && e < fetch.t1;
                const uint32_t pg = in ? pages[e >> a.c.shift] : PAGED_NONE;
                const bool ok = pg < a.c.pages;
                bad |= in && !ok;
                const unsigned char* src = ok ? srcK + pg * page_bytes + (e & in_page) * (HD * 2u) : a.c.k;
                const uint32_t to = (dst ^ ((c * ROWS_AT_ONCE & 7u) * 16u)) + c * (ROWS_AT_ONCE * HD * 2u);
                cp_async16_or_zero(to, src, ok ? 16u : 0u);
                cp_async16_or_zero(to + toSV, ok ? src + toV : a.c.v, ok ? 16u : 0u);
            }
        }
        if (paged_list_next(list, fetch, rows, units, SPAN) && f + 1u < count) aim();
    };
    aim();
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        if ((uint32_t)s < count) load(s);
        cp_async_commit();
    }

    // ldmatrix: the lane's row and 16-byte piece; the pieces of a product step follow by exclusive or
    const uint32_t mj = lane >> 3, kr = (mj >> 1) * 8 + (lane & 7u), vr = (mj & 1u) * 8 + (lane & 7u);
    const uint32_t k_at = ring + kr * (HD * 2u) + (((mj & 1u) ^ (kr & 7u)) * 16u);
    const uint32_t v_at = ring + toSV + vr * (HD * 2u) + (((mj >> 1) ^ (vr & 7u)) * 16u);
    constexpr int H = WIDE ? 2 : 1;  // heads of a thread
    uint32_t qa[KS][4], qb[WIDE ? KS : 1][4];
    float o[NT][4], m_run[H], l_run[H], down[H];  // scores are multiplied by down
    uint32_t head0 = 0, G = 0, tile_begin = 0;
    bool entering = true;
    for (uint32_t f = 0; f < count; ++f) {
        if (entering) {
            const uint32_t kvh = at.unit / subgroups, g0 = (at.unit - kvh * subgroups) * a.heads_at_once;
            G = min(a.heads_at_once, a.group - g0);
            head0 = kvh * a.group + g0;
            tile_begin = at.tile;
            // A operand of the scores: rows 0-7 hi, 8-15 lo of heads 0-7; WIDE: rows are heads, hi and lo apart
            const float* q0 = a.q + ((size_t)(row0 + at.row) * a.q_heads + head0 + g) * HD + 2 * t4;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                float2 x[KS][2];
                float big = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * KS; ++i) {
                    float2& y = x[i / 2][i % 2];
                    y = g + 8u * h < G ? *reinterpret_cast<const float2*>(q0 + 8 * HD * h + 8 * i) : make_float2(0.0f, 0.0f);
                    y.x *= a.scale, y.y *= a.scale;
                    big = fmaxf(big, fmaxf(fabsf(y.x), fabsf(y.y)));
                }
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                const uint32_t up = min(263u - (__float_as_uint(big) >> 23), 247u);
                const float factor = __uint_as_float(up << 23);
                down[h] = __uint_as_float((254u - up) << 23);
#pragma unroll
                for (int i = 0; i < 2 * KS; ++i) {
                    const float2 y = x[i / 2][i % 2];
                    const int at_a = 2 * (i % 2) + (WIDE ? h : 0);
                    uint32_t* lo_at = WIDE ? &qb[WIDE ? i / 2 : 0][at_a] : &qa[i / 2][at_a + 1];
                    split_h2(y.x * factor, y.y * factor, &qa[i / 2][at_a], lo_at);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
#pragma unroll
            for (int h = 0; h < H; ++h) m_run[h] = -INFINITY, l_run[h] = 0.0f;
        }
        cp_async_wait<STAGES - 2>();
        __syncthreads();
        // the stage that is filled again was read by products that have been issued: their operands are in registers
        if (f + STAGES - 1 < count) load(f + STAGES - 1);
        cp_async_commit();
        const uint32_t stage = (f % STAGES) * Cfg::STAGE;
        const uint32_t base = at.first + at.tile * SPAN + warp * TILE, e0 = base + 2 * t4;
        if (base < at.t1 && base + TILE > at.t0) {
        float s0[2][4], s1[2][4];  // even and odd product steps: two short chains each
#pragma unroll
        for (int i = 0; i < 4; ++i) s0[0][i] = s0[1][i] = s1[0][i] = s1[1][i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t b[4];
            ldmatrix_at(b, (k_at + stage) ^ (ks * 32u));
            mma16816(s0[ks & 1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b[0], b[1]);
            mma16816(s1[ks & 1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b[2], b[3]);
            if (WIDE) {
                mma16816(s0[ks & 1], qb[ks][0], qb[ks][1], qb[ks][2], qb[ks][3], b[0], b[1]);
                mma16816(s1[ks & 1], qb[ks][0], qb[ks][1], qb[ks][2], qb[ks][3], b[2], b[3]);
            }
        }
        // this thread's entries: e0, e0 + 1, e0 + 8, e0 + 9
        float s[H][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s0[0][i] += s0[1][i], s1[0][i] += s1[1][i];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            s[h][0] = WIDE ? s0[0][2 * h] : s0[0][0] + s0[0][2], s[h][1] = WIDE ? s0[0][2 * h + 1] : s0[0][1] + s0[0][3];
            s[h][2] = WIDE ? s1[0][2 * h] : s1[0][0] + s1[0][2], s[h][3] = WIDE ? s1[0][2 * h + 1] : s1[0][1] + s1[0][3];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[h][i] *= down[h];
        }
        if (base < at.t0 || base + TILE > at.t1 || __any_sync(0xffffffffu, bad)) {
            const uint32_t* own_pages = a.c.table + (size_t)list.slot[at.row] * a.c.max_pages;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t e = e0 + (i & 1) + (i >> 1) * 8;
                if (e < at.t0 || e >= at.t1 || own_pages[e >> a.c.shift] >= a.c.pages) {
#pragma unroll
                    for (int h = 0; h < H; ++h) s[h][i] = -INFINITY;
                }
            }
        }
        if (a.scores) {
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {  // entries outside the row's are not read again
                    const uint32_t e = e0 + 8u * i;
                    if (g + 8u * h < G && e < a.ld_scores)
                        *reinterpret_cast<float2*>(a.scores + ((size_t)(row0 + at.row) * a.q_heads + head0 + g + 8u * h) * a.ld_scores + e) =
                            make_float2(s[h][2 * i], s[h][2 * i + 1]);
                }
        }
        uint32_t ph[H][2], pl[H][2];
        bool moved = false;
        float corr[H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            float mx = fmaxf(fmaxf(s[h][0], s[h][1]), fmaxf(s[h][2], s[h][3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run[h], mx - WEIGHT_BIAS), use = m_new == -INFINITY ? 0.0f : m_new;
            moved |= m_new > m_run[h];
            corr[h] = fast_exp2(m_run[h] - use);
            const float p0 = fast_exp2(s[h][0] - use), p1 = fast_exp2(s[h][1] - use);
            const float p2 = fast_exp2(s[h][2] - use), p3 = fast_exp2(s[h][3] - use);
            l_run[h] = l_run[h] * corr[h] + ((p0 + p1) + (p2 + p3));  // this thread's entries; the quad's sums meet at the end
            m_run[h] = m_new;
            split_h2(p0, p1, &ph[h][0], &pl[h][0]);
            split_h2(p2, p3, &ph[h][1], &pl[h][1]);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                o[n][0] *= corr[0], o[n][1] *= corr[0];
                o[n][2] *= corr[H - 1], o[n][3] *= corr[H - 1];
            }
        }
#pragma unroll
        for (int nd = 0; nd < HD / 16; ++nd) {
            uint32_t b[4];
            ldmatrix_trans_at(b, (v_at + stage) ^ (nd * 32u));
            if (WIDE) {
                mma16816(o[2 * nd], ph[0][0], ph[H - 1][0], ph[0][1], ph[H - 1][1], b[0], b[1]);
                mma16816(o[2 * nd + 1], ph[0][0], ph[H - 1][0], ph[0][1], ph[H - 1][1], b[2], b[3]);
                mma16816(o[2 * nd], pl[0][0], pl[H - 1][0], pl[0][1], pl[H - 1][1], b[0], b[1]);
                mma16816(o[2 * nd + 1], pl[0][0], pl[H - 1][0], pl[0][1], pl[H - 1][1], b[2], b[3]);
            } else {
                mma16816(o[2 * nd], ph[0][0], pl[0][0], ph[0][1], pl[0][1], b[0], b[1]);
                mma16816(o[2 * nd + 1], ph[0][0], pl[0][0], ph[0][1], pl[0][1], b[2], b[3]);
            }
        }
        }
        const bool ends = at.tile + 1u == at.tiles;
        if (ends || f + 1u == count) {
            // this warp's part of the unit, for the join or (DIRECT) for this CTA
            const uint32_t row = row0 + at.row, kvh = at.unit / subgroups;
            const size_t part = (((size_t)at.row * units + at.unit + worker) * TILES_WARPS + warp) * a.heads_at_once;
            float* own_o = DIRECT ? warp_part(warp) : a.part_o + part * HD;
            float* own_m = DIRECT ? own_o + ROWS * HD : a.part_m + part;
            float* own_l = DIRECT ? own_m + ROWS : a.part_l + part;
            if (DIRECT) {
                cp_async_wait<0>();
                __syncthreads();  // the rings are done with
            }
            bool fine[H];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                float l = l_run[h];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                fine[h] = is_finite(l);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (!WIDE) o[n][0] += o[n][2], o[n][1] += o[n][3];
                    fine[h] &= is_finite(o[n][2 * h]) & is_finite(o[n][2 * h + 1]);
                }
                if (g + 8u * h < G) {
                    if (t4 == 0) own_m[g + 8 * h] = m_run[h], own_l[g + 8 * h] = l;
                    float* dst = own_o + (g + 8 * h) * HD + 2 * t4;
#pragma unroll
                    for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                }
            }
#pragma unroll
            for (int h = 0; h < H; ++h) {
                uint32_t odd = __ballot_sync(0xffffffffu, !fine[h] && g + 8u * h < G);
                while (odd) {  // a head with something that is not finite: again, in plain f32
                    const uint32_t gh = (__ffs(odd) - 1u) / 4u, head = head0 + gh + 8u * h;
                    odd &= ~(0xfu << (4u * gh));
                    const uint32_t own = gh + 8u * h;
                    const size_t at_head = (size_t)row * a.q_heads + head;
                    __syncwarp();
                    paged_plain_run<HD>(a, list.slot[at.row], kvh, a.q + at_head * HD, a.scores ? a.scores + at_head * a.ld_scores : nullptr,
                                          max(at.t0, at.first + tile_begin * SPAN), min(at.t1, at.first + (at.tile + 1u) * SPAN), warp, WEIGHT_BIAS, own_m + own, own_l + own,
                                          own_o + own * HD);
                }
            }
        }
        entering = paged_list_next(list, at, rows, units, SPAN);
    }
    cp_async_wait<0>();
    if (bad) atomicOr(a.status, 1u);
    if constexpr (DIRECT) {
        const uint32_t unit = worker - row0 * units, kvh = unit / subgroups, g0 = (unit - kvh * subgroups) * a.heads_at_once;
        G = min(a.heads_at_once, a.group - g0);
        const size_t first_head = (size_t)row0 * a.q_heads + kvh * a.group + g0;
        if (count == 0 && lane < ROWS) warp_part(warp)[ROWS * HD + lane] = -INFINITY, warp_part(warp)[ROWS * HD + ROWS + lane] = 0.0f;
        __syncthreads();
        // up to 8 parts with maximum m(i), sum l(i) and output o(i), in their order, all on their way first; a sum without a maximum stays NaN, as it is
        const auto join = [](auto most, uint32_t n, auto m, auto l, auto o, float* M_out, float* L_out) {
            constexpr uint32_t N = decltype(most)::value;
            float pm[N], pl[N], po[N], M = -INFINITY, L = 0.0f, O = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const bool in = i < n;
                pm[i] = in ? m(i) : -INFINITY, pl[i] = in ? l(i) : 0.0f, po[i] = in ? o(i) : 0.0f;
                M = fmaxf(M, pm[i]);
            }
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const float e = pl[i] != 0.0f ? (pm[i] == -INFINITY ? 1.0f : exp2f(pm[i] - M)) : 0.0f;
                L += pl[i] * e;
                if (e != 0.0f) O = fmaf(e, po[i], O);
            }
            *M_out = M, *L_out = L;
            return O;
        };
        const auto of_warps = [&](uint32_t i, float* M, float* L) {  // value i of the heads' outputs
            const uint32_t h = i / HD, d = i % HD;
            return join(std::integral_constant<uint32_t, TILES_WARPS>(), TILES_WARPS, [&](uint32_t w) { return warp_part(w)[ROWS * HD + h]; }, [&](uint32_t w) { return warp_part(w)[ROWS * HD + ROWS + h]; },
                        [&](uint32_t w) { return warp_part(w)[h * HD + d]; }, M, L);
        };
        const auto finish = [&](uint32_t i, float M, float L, float O) {
            const size_t head = first_head + i / HD;
            a.out[head * HD + i % HD] = L == 0.0f ? 0.0f : O / L;
            if (a.stat && i % HD == 0) a.stat[2 * head] = M == -INFINITY ? 0.0f : M, a.stat[2 * head + 1] = L == 0.0f ? 0.0f : 1.0f / L;
        };
        float M, L;
        if (peers == 1u) {
            for (uint32_t i = tid; i < G * HD; i += TILES_THREADS) {
                const float O = of_warps(i, &M, &L);
                finish(i, M, L, O);
            }
            return;
        }
        const uint32_t me = tc::cluster_rank(), slice = G * HD / peers;  // HD is a multiple of every cluster
        float* told_m = reinterpret_cast<float*>(smem + Cfg::SMEM);      // [peers][ROWS]
        float *told_l = told_m + DIRECT_CLUSTER * ROWS, *told_o = told_l + DIRECT_CLUSTER * ROWS;  // [peers][slice]
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (uint32_t i = tid; i < G * HD; i += TILES_THREADS) {
            const float O = of_warps(i, &M, &L);
            const uint32_t to = i / slice, h = i / HD;
            tc::st_cluster(tc::map_to_rank(tc::smem_u32(told_o + me * slice + i - to * slice), to), __float_as_uint(O));
            if (i % HD < peers) {  // one of them tells CTA i % HD
                tc::st_cluster(tc::map_to_rank(tc::smem_u32(told_m + me * ROWS + h), i % HD), __float_as_uint(M));
                tc::st_cluster(tc::map_to_rank(tc::smem_u32(told_l + me * ROWS + h), i % HD), __float_as_uint(L));
            }
        }
        __syncwarp();
        tc::cluster_sync_all();  // the last word between the CTAs: any may leave after it
        for (uint32_t j = tid; j < slice; j += TILES_THREADS) {
            const uint32_t i = me * slice + j, h = i / HD;
            const float O = join(std::integral_constant<uint32_t, DIRECT_CLUSTER>(), peers, [&](uint32_t c) { return told_m[c * ROWS + h]; }, [&](uint32_t c) { return told_l[c * ROWS + h]; },
                                 [&](uint32_t c) { return told_o[c * slice + j]; }, &M, &L);
            finish(i, M, L, O);
        }
    }
}

// The parts of one q head, put together in a fixed order by 256 threads: thread s has the weights of parts s, s + 256, .. (at most PAGED_PARTS_MOST);
// then 256 / LANES groups of lanes take every so-many-th part, each lane V dimensions, and the groups' sums meet in shared memory. CTAs of 8 lanes share a
// head's dimensions where there are few heads, for more loads at a time.
template <int V, int LANES, typename Part>
__device__ __forceinline__ void paged_join_parts(const PagedAttnArgs& a, size_t head, uint32_t share, uint32_t parts, Part part) {
    constexpr uint32_t MOST = PAGED_PARTS_MOST, GROUPS = 256 / LANES, AT_ONCE = 4;
    static_assert(MOST % 256u == 0, "a thread's parts");
    __shared__ float sw[MOST], red[16];
    __shared__ float s_acc[8][LANES * V];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, hd = a.c.hd;
    const uint32_t vl = tid % LANES, group = tid / LANES, d = (share * LANES + vl) * V;
    float x[AT_ONCE][V];
    const auto fetch = [&](uint32_t s0) {
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; ++k) {
            const uint32_t s = s0 + k * GROUPS;
            if (s >= parts || d >= hd) continue;
            const float* src = a.part_o + part(s) * hd + d;
            if constexpr (V == 4) {
                const float4 y = *reinterpret_cast<const float4*>(src);
                x[k][0] = y.x, x[k][1] = y.y, x[k][2] = y.z, x[k][3] = y.w;
            } else {
                x[k][0] = src[0];
            }
        }
    };
    fetch(group);  // on their way while the weights are made
    float m[MOST / 256], l[MOST / 256], M = -INFINITY, L = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < MOST / 256u; ++j) {
        const uint32_t s = tid + 256u * j;
        m[j] = -INFINITY, l[j] = 0.0f;
        if (256u * j >= parts) continue;
        if (s < parts) l[j] = a.part_l[part(s)], m[j] = a.part_m[part(s)];
        M = fmaxf(M, m[j]);  // an empty part's is -inf
    }
    M = warp_max(M);
    if (lane == 0) red[warp] = M;
    __syncthreads();
    M = red[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) M = fmaxf(M, red[i]);
#pragma unroll
    for (uint32_t j = 0; j < MOST / 256u; ++j) {
        if (256u * j >= parts) continue;
        const float e = l[j] != 0.0f ? (m[j] == -INFINITY ? 1.0f : exp2f(m[j] - M)) : 0.0f;  // a sum without a maximum: NaN, as it is
        sw[tid + 256u * j] = e;
        L += l[j] * e;
    }
    L = warp_sum(L);
    if (lane == 0) red[8 + warp] = L;
    __syncthreads();
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) L += red[8 + i];
    if (a.stat && tid == 0 && share == 0) a.stat[2 * head] = M == -INFINITY ? 0.0f : M, a.stat[2 * head + 1] = L == 0.0f ? 0.0f : 1.0f / L;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    for (uint32_t s0 = group; s0 < parts; s0 += AT_ONCE * GROUPS) {
        if (s0 != group) fetch(s0);
        if (d < hd)
#pragma unroll
            for (uint32_t k = 0; k < AT_ONCE; ++k) {
                const uint32_t s = s0 + k * GROUPS;
                const float w = s < parts ? sw[s] : 0.0f;
                if (w != 0.0f)  // an empty part's outputs may be anything
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] = fmaf(w, x[k][i], acc[i]);
            }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (lane < LANES)
#pragma unroll
        for (int i = 0; i < V; ++i) s_acc[warp][i * LANES + lane] = acc[i];
    __syncthreads();
    if (tid < LANES * V) {  // value tid: i = tid / LANES of lane tid % LANES
        const uint32_t at = (share * LANES + tid % LANES) * V + tid / LANES;
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) o += s_acc[w][tid];
        if (at < hd) a.out[head * hd + at] = L == 0.0f ? 0.0f : o / L;
    }
}

// Parts of paged_rows_kernel: [row][q head][split].
template <int V, int LANES>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedAttnArgs a) {
    pdl_wait();
    pdl_trigger();
    const size_t head = (size_t)blockIdx.y * a.q_heads + blockIdx.x, base = head * a.splits;
    paged_join_parts<V, LANES>(a, head, blockIdx.z, a.splits, [=](uint32_t s) { return base + s; });
}

// Of one q head of row r of a launch of `rows`: how many parts the warps left, and where. Nothing for a row without entries.
struct PagedParts {
    uint32_t n, first, h;
    __device__ __forceinline__ size_t at(const PagedAttnArgs& a, uint32_t s) const { return ((size_t)first + s) * a.heads_at_once + h; }
};
struct PagedBefore {  // tiles before the row, before the next one, of all rows
    uint64_t row, next, all;
};
__device__ __forceinline__ PagedBefore paged_before(const PagedAttnArgs& a, uint32_t r, uint32_t rows) {
    return PagedBefore{a.prefix[r], a.prefix[r + 1], a.prefix[rows]};
}
__device__ __forceinline__ PagedParts paged_parts(const PagedAttnArgs& a, uint32_t r, const PagedBefore& b, uint32_t q_head) {
    const uint32_t kvh = q_head / a.group, in_group = q_head - kvh * a.group;
    const uint32_t subgroups = (a.group + a.heads_at_once - 1u) / a.heads_at_once, units = a.c.kv_heads * subgroups;
    const uint32_t unit = kvh * subgroups + in_group / a.heads_at_once;
    const uint64_t before = b.row, tiles = b.next - before, total = b.all * units;
    if (tiles == 0) return PagedParts{0u, 0u, 0u};
    const uint32_t n = ctas_at_work(total, a.workers);
    const uint64_t lo = before * units + unit * tiles;
    const uint32_t w0 = cta_of(lo, total, n), w1 = cta_of(lo + tiles - 1u, total, n);
    return PagedParts{(w1 - w0 + 1u) * a.part_warps, (r * units + unit + w0) * a.part_warps, in_group % a.heads_at_once};
}

// Parts of paged_tiles_kernel and paged_lanes_kernel, and the zeros of rows without entries: a q head of row r, a share of the dimensions.
template <int LANES>
__device__ __forceinline__ void paged_join_head(const PagedAttnArgs& a, uint32_t r, uint32_t rows, uint32_t q_head, uint32_t share) {
    const size_t head = (size_t)(a.row0 + r) * a.q_heads + q_head;
    const PagedParts parts = paged_parts(a, r, paged_before(a, r, rows), q_head);
    if (parts.n == 0) {
        if (share == 0)
            for (uint32_t d = threadIdx.x; d < a.c.hd; d += 256u) a.out[head * a.c.hd + d] = 0.0f;
        return;
    }
    paged_join_parts<4, LANES>(a, head, share, parts.n, [&](uint32_t s) { return parts.at(a, s); });
}
// Grid (q head, row of the launch, share of the dimensions).
template <int LANES>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedAttnArgs a) {
    pdl_wait();
    pdl_trigger();
    paged_join_head<LANES>(a, blockIdx.y, gridDim.y, blockIdx.x, blockIdx.z);
}

// A head's maximum and 1 / sum from its parts, by a warp: what paged_join_parts leaves in a.stat.
__device__ __forceinline__ float2 paged_parts_stat(const PagedAttnArgs& a, const PagedParts& parts) {
    float M = -INFINITY, L = 0.0f;
#pragma unroll 1
    for (uint32_t s = threadIdx.x & 31u; s < parts.n; s += 32u) {
        const float l = a.part_l[parts.at(a, s)], m = a.part_m[parts.at(a, s)];
        const float top = fmaxf(M, m), use = top == -INFINITY ? 0.0f : top;  // a sum without a maximum: NaN, as it is
        L = (M == -INFINITY ? L : L * exp2f(M - use)) + (l == 0.0f ? 0.0f : (m == -INFINITY ? l : l * exp2f(m - use)));
        M = top;
    }
    const float top = warp_max(M);
    L = warp_sum(M == -INFINITY ? L : L * exp2f(M - top));
    return make_float2(top == -INFINITY ? 0.0f : top, L == 0.0f ? 0.0f : 1.0f / L);
}

// CTA = (1024 entries, kv head, row); only the first row of a slot works, for all rows of the slot in their order, so that sums do not
// depend on who comes first. Thread = four neighbouring entries (one after the other where weights or scores are not 16-byte aligned).
// PARTS: the statistics come from the parts, not from a.stat. Bound by the chain rows, parts and scores, weights.
constexpr uint32_t WEIGHTS_AT_ONCE = 1024, WEIGHTS_GROUP = 64, WEIGHTS_HEADS = 4;
template <bool PARTS>
__device__ __forceinline__ void paged_weights(const PagedAttnArgs& a, uint32_t vec, uint32_t piece, uint32_t h, uint32_t row) {
    __shared__ float2 s_stat[PARTS ? WEIGHTS_GROUP : 1];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, e0 = piece * WEIGHTS_AT_ONCE, e = e0 + 4u * tid;
    float4 x[WEIGHTS_HEADS];  // scores of up to four heads
    const auto fetch = [&](size_t head, uint32_t g0, uint32_t to) {
#pragma unroll
        for (uint32_t g = 0; g < WEIGHTS_HEADS; ++g)
            if (g0 + g < a.group && e < to) x[g] = *reinterpret_cast<const float4*>(a.scores + (head + g0 + g) * a.ld_scores + e);
    };
    PagedBefore tiles_before{};
    if (PARTS) tiles_before = paged_before(a, row, a.rows);
    const uint32_t slot = a.row_slot[row];
    if (slot >= a.c.slots) return;
    // every warp looks at all rows, 32 at a time, a lane each
    uint32_t s, b, n, most = 0;
    bool skip = false;
    for (uint32_t r0 = 0; r0 < a.rows; r0 += 32u) {
        const uint32_t r = r0 + lane;
        const bool inside = r < a.rows && paged_row_range(a, r, &s, &b, &n), mine = r < a.rows && s == slot;
        if (mine) skip |= r < row || !inside, most = max(most, n);
    }
    if (__any_sync(0xffffffffu, skip)) return;
    most = __reduce_max_sync(0xffffffffu, most);
    if (e0 >= most) return;
    const size_t at = ((size_t)slot * a.c.kv_heads + h) * a.ld_weights + e;
    const bool whole = vec && e + 4u <= most;
    float w[4];
    if (whole && a.weights_in) {
        const float4 y = *reinterpret_cast<const float4*>(a.weights_in + at);
        w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) w[i] = a.weights_in && e + i < most ? a.weights_in[at + i] : 0.0f;
    }
    for (uint32_t r0 = row & ~31u; r0 < a.rows; r0 += 32u) {
        const uint32_t r = r0 + lane;
        if (a.rows > 32u && r < a.rows) paged_row_range(a, r, &s, &b, &n);  // up to 32 are there already
        uint32_t mask = __ballot_sync(0xffffffffu, r < a.rows && s == slot);
        while (mask) {  // the slot's rows in order, `row` the first
            const uint32_t k = __ffs(mask) - 1u, from = __shfl_sync(0xffffffffu, b, k), to = __shfl_sync(0xffffffffu, n, k), now = r0 + k;
            mask &= mask - 1u;
            if (from >= to || e0 >= to || e0 + WEIGHTS_AT_ONCE <= from) continue;  // the same for all threads
            const size_t head = (size_t)now * a.q_heads + h * a.group;
            fetch(head, 0u, to);  // on their way while the statistics are made
            if constexpr (PARTS) {
                __syncthreads();
                const PagedBefore before = now == row ? tiles_before : paged_before(a, now, a.rows);
                for (uint32_t g = tid >> 5; g < a.group; g += 8u) {
                    const float2 y = paged_parts_stat(a, paged_parts(a, now, before, h * a.group + g));
                    if (lane == 0) s_stat[g] = y;
                }
                __syncthreads();
            }
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t g0 = 0; g0 < a.group; g0 += WEIGHTS_HEADS) {
                if (g0) fetch(head, g0, to);
#pragma unroll
                for (uint32_t j = 0; j < WEIGHTS_HEADS; ++j) {
                    const uint32_t g = g0 + j;
                    if (g >= a.group) break;
                    const float M = PARTS ? s_stat[g].x : a.stat[2 * (head + g)], inv = PARTS ? s_stat[g].y : a.stat[2 * (head + g) + 1];
                    sum[0] += e >= from && e < to ? exp2f(x[j].x - M) * inv : 0.0f;
                    sum[1] += e + 1u >= from && e + 1u < to ? exp2f(x[j].y - M) * inv : 0.0f;
                    sum[2] += e + 2u >= from && e + 2u < to ? exp2f(x[j].z - M) * inv : 0.0f;
                    sum[3] += e + 3u >= from && e + 3u < to ? exp2f(x[j].w - M) * inv : 0.0f;
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) w[i] += sum[i];
        }
    }
    if (whole) {
        *reinterpret_cast<float4*>(a.weights_out + at) = make_float4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (e + i < most) a.weights_out[at + i] = w[i];
    }
}
__global__ void __launch_bounds__(256) paged_weights_kernel(PagedAttnArgs a, uint32_t vec) {
    pdl_wait();
    pdl_trigger();
    paged_weights<false>(a, vec, blockIdx.x, blockIdx.y, blockIdx.z);
}
// Weights and join side by side: `weighing` CTAs of paged_weights (piece of the entries, kv head, row), which look at the parts themselves instead of waiting for
// the join, then those of the join (q head, row, share). All rows are in one launch. Us of the whole call against one after the other: 12 rows of 509 to
// 8192 entries, 32 / 8 heads of 128, 53.4 (55.9), one of 8192 18.6 (19.9), 60 of 500 to 3000 103 (103), 9 of f32 24.5 (27.8). 64 registers, and the parts one by one: with
// four of them at a time 56.3, with 85 registers 53.5 and 106, with 51 55.4 and 106.
template <int LANES>
__global__ void __launch_bounds__(256, 4) paged_join_weights_kernel(PagedAttnArgs a, uint32_t vec, uint32_t weighing, uint32_t pieces) {
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x < weighing) {
        const uint32_t x = blockIdx.x / pieces, row = x / a.c.kv_heads;
        paged_weights<true>(a, vec, blockIdx.x - x * pieces, x - row * a.c.kv_heads, row);
    } else {
        const uint32_t b = blockIdx.x - weighing, x = b / a.q_heads, share = x / a.rows;
        paged_join_head<LANES>(a, x - share * a.rows, a.rows, b - x * a.q_heads, share);
    }
}

// Whether a CTA per head and row leaves most of the device idle.
bool few_heads(const M40llmCudaContext* ctx, uint32_t q_heads, uint32_t rows) { return (uint64_t)q_heads * rows <= 2ull * (uint64_t)ctx->sm_count; }

template <int HD, bool WIDE, bool DIRECT>
cudaError_t launch_tiles(M40llmCudaContext* ctx, const PagedAttnArgs& a, uint32_t peers) {
    using Cfg = TilesCfg<HD, WIDE>;
    constexpr int smem = Cfg::SMEM + (DIRECT ? Cfg::TOLD : 0);
    const cudaError_t e = cudaFuncSetAttribute(paged_tiles_kernel<HD, WIDE, DIRECT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.workers * peers);
    cfg.blockDim = dim3(TILES_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->decode_stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = m40_pdl_enabled() ? attr : attr + 1;
    cfg.numAttrs = m40_pdl_enabled() ? 1 : 0;
    if (peers > 1u) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = peers;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    return cudaLaunchKernelEx(&cfg, paged_tiles_kernel<HD, WIDE, DIRECT>, a);
}
template <bool DIRECT>
cudaError_t launch_tiles_of(M40llmCudaContext* ctx, const PagedAttnArgs& a, uint32_t peers) {
    const bool wide = a.heads_at_once > 8u;
    if (a.c.hd == 64u) return wide ? launch_tiles<64, true, DIRECT>(ctx, a, peers) : launch_tiles<64, false, DIRECT>(ctx, a, peers);
    return wide ? launch_tiles<128, true, DIRECT>(ctx, a, peers) : launch_tiles<128, false, DIRECT>(ctx, a, peers);
}

// All rows in launches of up to 256, each followed by its join. `ctas`: how many are resident, `span`: entries of a tile of the list.
template <typename Launch>
cudaError_t launch_list(M40llmCudaContext* ctx, PagedAttnArgs a, uint32_t ctas, uint32_t span, uint32_t vec, bool* weighed, Launch launch) {
    const uint64_t most = (uint64_t)a.c.kv_heads * ((a.group + a.heads_at_once - 1u) / a.heads_at_once) * ((a.bound + span - 1u) / span) * a.rows;
    a.workers = most < ctas ? (uint32_t)most : ctas;
    cudaError_t e = cudaSuccess;
    const bool few = few_heads(ctx, a.q_heads, a.rows);
    const uint32_t pieces = (a.bound + WEIGHTS_AT_ONCE - 1u) / WEIGHTS_AT_ONCE;
    const uint64_t joins = (uint64_t)a.q_heads * a.rows * (few ? (a.c.hd + 31u) / 32u : (a.c.hd + 127u) / 128u);
    const uint64_t weighing = (uint64_t)pieces * a.c.kv_heads * a.rows, both = joins + weighing;
    *weighed = a.scores && a.rows <= LIST_ROWS && a.group <= WEIGHTS_GROUP && both <= 0x7fffffffu;
    if (*weighed) {
        e = launch(a);
        if (e == cudaSuccess)
            e = m40_launch_dependent(few ? paged_join_weights_kernel<8> : paged_join_weights_kernel<32>, dim3((uint32_t)both), dim3(256), 0, ctx->decode_stream, a, vec,
                                     (uint32_t)weighing, pieces);
        M40_COUNT_LAUNCH(ctx);
        M40_COUNT_LAUNCH(ctx);
        return e;
    }
    for (a.row0 = 0; e == cudaSuccess && a.row0 < a.rows; a.row0 += LIST_ROWS) {
        const uint32_t rows = a.rows - a.row0 < LIST_ROWS ? a.rows - a.row0 : LIST_ROWS, hd = a.c.hd;
        e = launch(a);
        if (e == cudaSuccess)
            e = few_heads(ctx, a.q_heads, rows)
                    ? m40_launch_dependent(paged_join_kernel<8>, dim3(a.q_heads, rows, (hd + 31u) / 32u), dim3(256), 0, ctx->decode_stream, a)
                    : m40_launch_dependent(paged_join_kernel<32>, dim3(a.q_heads, rows, (hd + 127u) / 128u), dim3(256), 0, ctx->decode_stream, a);
        M40_COUNT_LAUNCH(ctx);
        M40_COUNT_LAUNCH(ctx);
    }
    return e;
}

template <typename ET, int GT>
cudaError_t launch_rows(const PagedAttnArgs& a, dim3 grid, uint32_t T, uint32_t vec, uint32_t pitch, size_t smem, cudaStream_t s) {
    const uint32_t dv = (a.c.hd + ROWS_THREADS - 1) / ROWS_THREADS;
    void (*kernel)(PagedAttnArgs, uint32_t, uint32_t, uint32_t) =
        dv == 1 ? paged_rows_kernel<ET, GT, 1> : (dv == 2 ? paged_rows_kernel<ET, GT, 2> : paged_rows_kernel<ET, GT, 4>);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PAGED_SMEM_MOST);  // the same from every thread
    if (e != cudaSuccess) return e;
    return m40_launch_dependent(kernel, grid, dim3(ROWS_THREADS), smem, s, a, T, vec, pitch);
}

}  // namespace

extern "C" int m40llm_attention_paged_async(M40llmCudaContext* ctx, const M40llmPagedCache* cache, const M40llmPagedAttention* c) {
    if (!ctx || !cache || !c || !c->q || !c->out || !c->row_slot || !c->row_len) return -1;
    PagedAttnArgs a = {};
    const int rc = m40_paged_view(cache, &a.c);
    if (rc != 0) return rc;
    const uint32_t capacity = paged_capacity(a.c), hd = cache->head_dim;
    if (c->rows == 0 || c->q_heads == 0 || c->q_heads % cache->kv_heads != 0 || c->max_len > capacity) return -2;
    if (c->weights_out && c->ld_weights < capacity) return -2;
    const uint32_t bound = c->max_len ? c->max_len : capacity;
    const size_t heads = (size_t)c->rows * c->q_heads;
    // beside the scores, what the parts of fewer than 2^32 rows and heads take is below 2^52 bytes
    if (c->rows > 65535u || c->q_heads > 65535u || (c->weights_out && heads * bound > PAGED_SCRATCH_MOST / 8u)) return M40LLM_ERR_LIMIT;
    if (m40_ensure_device(ctx) != 0) return -1;
    a.q = (const float*)c->q;
    a.out = (float*)c->out;
    a.row_slot = c->row_slot;
    a.row_len = c->row_len;
    a.row_begin = c->row_begin;
    a.weights_in = (const float*)c->weights_in;
    a.weights_out = (float*)c->weights_out;
    a.status = ctx->d_status;
    a.rows = c->rows;
    a.q_heads = c->q_heads;
    a.group = c->q_heads / cache->kv_heads;
    a.ld_weights = c->ld_weights;
    a.bound = bound;
    a.scale = c->scale * LOG2E;
    cudaStream_t s = ctx->decode_stream;
    const bool f32 = cache->elem_dtype == M40LLM_DT_F32;
    const uint32_t vec = m40_paged_vec16(cache) ? 1u : 0u;
    const bool tiles = !f32 && vec && (hd == 64u || hd == 128u) && (((uintptr_t)c->q) & 7u) == 0;
    PagedLanes lanes = {};
    const bool by_lanes = !tiles && (((uintptr_t)c->q) & 15u) == 0 && m40_paged_lanes(ctx, cache, a.group, &lanes), list = tiles || by_lanes;
    // heads of a group in equal shares of up to 16; 8 take one product where 9 to 16 take two
    const uint32_t shares = (a.group + 15u) / 16u;
    a.heads_at_once = by_lanes ? lanes.heads_at_once : (a.group + shares - 1u) / shares;
    a.part_warps = by_lanes ? lanes.warps : TILES_WARPS;
    const uint32_t ctas = by_lanes ? lanes.ctas : paged_list_ctas((uint32_t)ctx->sm_count, hd == 64u ? TilesCfg<64, false>::CTAS : TilesCfg<128, false>::CTAS, TILES_WARPS);
    if (!list) {
        const uint64_t work = (uint64_t)c->rows * cache->kv_heads * a.bound, target = 2ull * (uint64_t)ctx->sm_count;
        uint64_t chunk = (work + target - 1) / target;
        chunk = chunk < 128u ? 128u : (chunk > 1024u ? 1024u : chunk);
        chunk = (chunk + 63u) & ~63ull;
        if ((a.bound + chunk - 1) / chunk > 256u) chunk = ((a.bound + 255u) / 256u + 63u) & ~63ull;
        a.chunk = (uint32_t)chunk;
        a.splits = (uint32_t)((a.bound + chunk - 1) / chunk);
    }
    const size_t units = (size_t)cache->kv_heads * ((a.group + a.heads_at_once - 1u) / a.heads_at_once);
    // Short rows: clusters of up to 8 CTAs that fill half of the device take a unit each, without a list and a join. How many tiles a CTA may have then: 32
    // with a wave of CTAs or more, 16 with half of one (the list deals uneven rows better, but its parts and their join cost more the more rows there are), else 4
    // (the list has more CTAs at work). Us, this against the list: one row of 64 / 700 / 2000 entries, 32 / 4 heads of 64, 4.9 / 6.7 / 8.3 against 6.9 / 7.5 / 8.2;
    // rows of 32 / 8 heads of 128: 4 of 1000 9.3 (11.0), 8 of up to 500 9.0 (11.8), 8 of 4000 29 (35), 8 of 8000 54.6 (54.7), 32 of 100 to 1000 23.5 (27.3),
    // 32 of 100 to 2000 38.7 (39.7), 200 of 100 to 500 65 (90), 200 of 100 to 2000 152 (182), 100 of 100 to 4000 160 (159). Clusters of 16 are not placed as they
    // come free: 2 rows of 1000 14.2 against 8.4 with 8. (In paged_lanes_kernel the list is
    // as fast or faster: 4 rows of up to 250 f32 entries 8.6 and 8.6, one of 700 11.1 against 8.2.)
    uint32_t peers = 1u;
    while (peers < DIRECT_CLUSTER && a.bound > SPAN * peers && (uint64_t)c->rows * units * peers * 2u <= ctas) peers *= 2u;
    const uint64_t direct_ctas = (uint64_t)c->rows * units * peers;
    const uint32_t most_tiles = direct_ctas >= ctas ? 32u : (2u * direct_ctas >= ctas ? 16u : 4u);
    const bool direct = tiles && a.bound <= SPAN * peers * most_tiles && direct_ctas <= 0x7fffffffu;
    const uint32_t span = by_lanes ? 8u * lanes.warps : SPAN;
    if (list && !direct && !paged_list_fits(c->rows < LIST_ROWS ? c->rows : LIST_ROWS, units, (a.bound + span - 1u) / span, ctas)) return M40LLM_ERR_LIMIT;
    if ((list && !direct) || a.splits > 1 || c->weights_out) {
        a.ld_scores = c->weights_out ? (a.bound + 3u) & ~3u : 0u;
        const size_t rows_at_once = c->rows < LIST_ROWS ? c->rows : LIST_ROWS;
        const size_t parts = direct ? 0 : (list ? (rows_at_once * units + ctas) * a.part_warps * a.heads_at_once : heads * a.splits);
        const size_t floats = parts * (hd + 2) + heads * 2 + 4 + heads * (size_t)a.ld_scores;
        const size_t prefix = (LIST_ROWS + 1) * sizeof(uint64_t);  // first, for its alignment; 16 bytes more keep the outputs' rows aligned
        unsigned char* work_area = (unsigned char*)m40_ensure_scratch(ctx, 1, prefix + 8 + floats * sizeof(float), 0);
        if (!work_area) return -5;
        a.prefix = (uint64_t*)work_area;
        a.part_o = (float*)(work_area + prefix + 8);
        a.part_m = a.part_o + parts * hd;
        a.part_l = a.part_m + parts;
        if (c->weights_out) {
            a.stat = a.part_l + parts;
            a.scores = a.part_o + ((parts * (hd + 2) + heads * 2 + 3) & ~(size_t)3);  // 16-byte aligned
        }
    }
    const bool aligned = ((((uintptr_t)a.weights_in) | ((uintptr_t)a.weights_out) | ((uintptr_t)a.scores)) & 15u) == 0 && a.ld_weights % 4u == 0;
    const uint32_t vec_weights = aligned ? 1u : 0u;
    bool weighed = false;
    cudaError_t e;
    if (direct) {
        a.workers = (uint32_t)(c->rows * units);
        e = launch_tiles_of<true>(ctx, a, peers);
        M40_COUNT_LAUNCH(ctx);
    } else if (tiles) {
        e = launch_list(ctx, a, ctas, span, vec_weights, &weighed, [&](const PagedAttnArgs& x) { return launch_tiles_of<false>(ctx, x, 1u); });
    } else if (by_lanes) {
        e = launch_list(ctx, a, ctas, span, vec_weights, &weighed, [&](const PagedAttnArgs& x) { return m40_paged_lanes_launch(ctx, x, lanes, f32); });
    } else {
        const uint32_t elem = f32 ? 4u : 2u, hd4 = (hd + 3u) & ~3u;
        const uint32_t T = hd4 * elem > 1024u ? 16u : 32u, pitch = ((hd4 * elem + 15u) & ~15u) / elem + 16u / elem;
        const uint32_t gt = a.group >= 8u ? 8u : (a.group >= 4u ? 4u : (a.group >= 2u ? 2u : 1u)), subgroups = (a.group + gt - 1) / gt;
        const dim3 grid(a.splits, cache->kv_heads * subgroups, c->rows);
        if (grid.y > 65535u) return M40LLM_ERR_LIMIT;
        const size_t smem = ((size_t)gt * hd4 + ROWS_THREADS * gt + gt * 32u + 8u + 64u) * 4u + 4ull * T * pitch * elem;
        if (f32)
            e = gt == 8   ? launch_rows<float, 8>(a, grid, T, vec, pitch, smem, s)
                : gt == 4 ? launch_rows<float, 4>(a, grid, T, vec, pitch, smem, s)
                : gt == 2 ? launch_rows<float, 2>(a, grid, T, vec, pitch, smem, s)
                          : launch_rows<float, 1>(a, grid, T, vec, pitch, smem, s);
        else
            e = gt == 8   ? launch_rows<__half, 8>(a, grid, T, vec, pitch, smem, s)
                : gt == 4 ? launch_rows<__half, 4>(a, grid, T, vec, pitch, smem, s)
                : gt == 2 ? launch_rows<__half, 2>(a, grid, T, vec, pitch, smem, s)
                          : launch_rows<__half, 1>(a, grid, T, vec, pitch, smem, s);
        M40_COUNT_LAUNCH(ctx);
        if (e == cudaSuccess && (a.splits > 1 || a.scores)) {
            if (hd % 4u != 0)
                e = m40_launch_dependent(paged_merge_kernel<1, 32>, dim3(c->q_heads, c->rows, (hd + 31u) / 32u), dim3(256), 0, s, a);
            else if (few_heads(ctx, c->q_heads, c->rows))
                e = m40_launch_dependent(paged_merge_kernel<4, 8>, dim3(c->q_heads, c->rows, (hd + 31u) / 32u), dim3(256), 0, s, a);
            else
                e = m40_launch_dependent(paged_merge_kernel<4, 32>, dim3(c->q_heads, c->rows, (hd + 127u) / 128u), dim3(256), 0, s, a);
            M40_COUNT_LAUNCH(ctx);
        }
    }
    if (e == cudaSuccess && a.scores && !weighed) {
        e = m40_launch_dependent(paged_weights_kernel, dim3((a.bound + WEIGHTS_AT_ONCE - 1u) / WEIGHTS_AT_ONCE, cache->kv_heads, c->rows), dim3(256), 0, s, a,
                                 vec_weights);
        M40_COUNT_LAUNCH(ctx);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        return -3;
    }
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
