// Attention of single tokens over a paged cache in f32 multiply-adds: caches of f32 entries, and f16 ones of head sizes that the tiles of
// attention_paged.cu do not take.
#include "attention_paged.cuh"
#include "stack_math.cuh"

namespace {

using namespace attn_mma;

constexpr uint32_t LANES_TILE = 8, LANES_STAGES = 3;  // entries of a warp's tile
// Where the warps' rings begin: behind their weights (doubled) and corrections, on 16 bytes, as copies want it.
__host__ __device__ constexpr uint32_t lanes_rings(uint32_t warps, uint32_t gt) { return (warps * (LANES_TILE * gt * 8u + gt * 4u) + 15u) & ~15u; }

__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 of_pair(uint64_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// four neighbouring elements as two pairs
__device__ __forceinline__ void load4(const float* p, uint64_t* r) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(p);
    r[0] = x.x, r[1] = x.y;
}
__device__ __forceinline__ void load4(const __half* p, uint64_t* r) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
    r[0] = pair_of(a.x, a.y), r[1] = pair_of(b.x, b.y);
}
__device__ __forceinline__ float xor_sum(float keep, float send, int mask) { return keep + __shfl_xor_sync(0xffffffffu, send, mask); }

// A run of the list of work per CTA, tiles of 8 entries per warp, which arrive by cp.async in a ring of three. GT q heads of a kv head at a time.
//   scores   lane = (16 slices of the dimensions, 2 halves of the tile): the slice's part of the queries stays in registers, and each key piece is read from
//            shared memory once for all heads. The 4 GT sums of a lane are added up over the slices by exchanges that halve them; a lane takes its entries
//            and heads in an order turned by its own number, so that what it keeps always comes first and nothing is selected. It ends with one entry and
//            GT / 4 heads (GT 2: one).
//   softmax  online in base 2, over the lanes with the same head.
//   outputs  lane = four neighbouring dimensions (DV times); weights come from shared memory, doubled, for two multiply-adds an instruction.
// hd <= 64 DQ = 128 DV. Bound by HBM. Against 32-entry tiles for the CTA with four barriers each (paged_rows_kernel): 9 rows of up to 4097 f32 entries
// 46.5 -> 20.0 us.
template <typename ET, int GT, int DQ>
__global__ void __launch_bounds__(256, 1) paged_lanes_kernel(PagedAttnArgs a) {
    constexpr int DV = DQ / 2, HPL = GT == 8 ? 2 : 1;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ PagedList list;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, warps = blockDim.x / 32u, span = LANES_TILE * warps;
    const uint32_t hd = a.c.hd, rb = hd * (uint32_t)sizeof(ET), tile_bytes = LANES_TILE * rb;
    // the warp's memory: weights [8][GT] doubled, corrections [GT], then the ring: K and V of a stage after each other
    float2* s_p = reinterpret_cast<float2*>(smem) + warp * (LANES_TILE * GT);
    float* s_corr = reinterpret_cast<float*>(smem + warps * (LANES_TILE * GT * 8u)) + warp * GT;
    unsigned char* ring = smem + lanes_rings(warps, GT) + warp * (LANES_STAGES * 2u * tile_bytes);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const uint32_t units = a.c.kv_heads * ((a.group + a.heads_at_once - 1u) / a.heads_at_once), subgroups = units / a.c.kv_heads;
    const uint32_t rows = min(a.rows - a.row0, LIST_ROWS);
    pdl_wait();
    pdl_trigger();
    if (warp == 0) paged_list_make(a, list, rows, span);
    __syncthreads();
    const uint64_t total = list.prefix[rows] * units;
    const uint32_t worker = blockIdx.x, workers = ctas_at_work(total, a.workers);
    if (worker >= workers) return;
    const uint64_t lo = quotient(worker * total, workers);
    const uint32_t count = (uint32_t)(quotient((worker + 1u) * total, workers) - lo);  // at least 1
    PagedPlace at = paged_list_at(list, lo, rows, units, span), fetch = at;

    const uint32_t in_page = (1u << a.c.shift) - 1u, pieces = rb / 16u;
    const uint64_t head_bytes = (uint64_t)rb << a.c.shift, page_bytes = a.c.kv_heads * head_bytes;
    const ptrdiff_t toV = a.c.v - a.c.k;
    bool bad = false;  // the warp met a page outside the pool
    const auto load = [&](uint32_t f) {
        const uint32_t base = fetch.first + fetch.tile * span + warp * LANES_TILE, dst = ring_at + (f % LANES_STAGES) * 2u * tile_bytes;
        const uint32_t* pages = a.c.table + (size_t)list.slot[fetch.row] * a.c.max_pages;
        const unsigned char* srcK = a.c.k + fetch.unit / subgroups * head_bytes;
        if (a.c.shift >= 3u && base >= fetch.t0 && base + LANES_TILE <= fetch.t1) {  // a whole tile, one run of memory
            const uint32_t pg = pages[base >> a.c.shift];
            const bool ok = pg < a.c.pages;
            bad |= !ok;
            const unsigned char* src = srcK + (ok ? pg * page_bytes : 0) + (size_t)(base & in_page) * rb;
#pragma unroll 4
            for (uint32_t p = lane; p < LANES_TILE * pieces; p += 32u) {
                cp_async16_or_zero(dst + p * 16u, src + p * 16u, ok ? 16u : 0u);
                cp_async16_or_zero(dst + tile_bytes + p * 16u, src + toV + p * 16u, ok ? 16u : 0u);
            }
        } else if (base < fetch.t1 && base + LANES_TILE > fetch.t0) {
            for (uint32_t p = lane; p < LANES_TILE * pieces; p += 32u) {
                const uint32_t r = p / pieces, e = base + r;
                const bool in = e >= fetch.t0 && e < fetch.t1;
                const uint32_t pg = in ? pages[e >> a.c.shift] : PAGED_NONE;
                const bool ok = pg < a.c.pages;
                bad |= in && !ok;
                const unsigned char* src = ok ? srcK + pg * page_bytes + (size_t)(e & in_page) * rb + (p - r * pieces) * 16u : a.c.k;
                cp_async16_or_zero(dst + p * 16u, src, ok ? 16u : 0u);
                cp_async16_or_zero(dst + tile_bytes + p * 16u, ok ? src + toV : a.c.v, ok ? 16u : 0u);
            }
        }
        paged_list_next(list, fetch, rows, units, span);
    };
#pragma unroll
    for (uint32_t s = 0; s < LANES_STAGES - 1; ++s) {
        if (s < count) load(s);
        cp_async_commit();
    }

    const uint32_t slice = lane & 15u, half = lane >> 4, turn = slice & 3u, head_turn = slice >> 2;
    // the head that this lane's accumulator j belongs to
    const auto head_of = [&](uint32_t j) { return GT == 8 ? j ^ (head_turn << 1) : (GT == 4 ? j ^ head_turn : j ^ (head_turn & 1u)); };
    uint64_t q[GT][2 * DQ], acc[GT][2 * DV];
    float m_run[HPL], l_run[HPL];
    uint32_t head0 = 0, G = 0;
    bool entering = true;
    for (uint32_t f = 0; f < count; ++f) {
        if (entering) {
            const uint32_t kvh = at.unit / subgroups, g0 = (at.unit - kvh * subgroups) * a.heads_at_once;
            G = min(a.heads_at_once, a.group - g0);
            head0 = kvh * a.group + g0;
            const float* q0 = a.q + ((size_t)(a.row0 + at.row) * a.q_heads + head0) * hd;
#pragma unroll
            for (uint32_t j = 0; j < GT; ++j)
#pragma unroll
                for (uint32_t i = 0; i < DQ; ++i) {
                    const uint32_t d = (slice + 16u * i) * 4u, h = head_of(j);
                    const float4 x = h < G && d < hd ? *reinterpret_cast<const float4*>(q0 + (size_t)h * hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                    q[j][2 * i] = pair_of(x.x * a.scale, x.y * a.scale), q[j][2 * i + 1] = pair_of(x.z * a.scale, x.w * a.scale);
                }
#pragma unroll
            for (uint32_t j = 0; j < GT; ++j)
#pragma unroll
                for (uint32_t i = 0; i < 2 * DV; ++i) acc[j][i] = 0u;
#pragma unroll
            for (int h = 0; h < HPL; ++h) m_run[h] = -INFINITY, l_run[h] = 0.0f;
        }
        cp_async_wait<LANES_STAGES - 2>();
        __syncwarp();
        if (f + LANES_STAGES - 1u < count) load(f + LANES_STAGES - 1u);
        cp_async_commit();
        const uint32_t base = at.first + at.tile * span + warp * LANES_TILE;
        if (base < at.t1 && base + LANES_TILE > at.t0) {
            const ET* tK = reinterpret_cast<const ET*>(ring + (f % LANES_STAGES) * 2u * tile_bytes);
            const ET* tV = reinterpret_cast<const ET*>(ring + (f % LANES_STAGES) * 2u * tile_bytes + tile_bytes);
            float x[4][GT];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const ET* kr = tK + (half * 4u + (i ^ turn)) * hd;
                uint64_t s[GT];
#pragma unroll
                for (uint32_t c = 0; c < DQ; ++c) {
                    const uint32_t d = (slice + 16u * c) * 4u;
                    uint64_t k[2] = {0u, 0u};
                    if (d < hd) load4(kr + d, k);
#pragma unroll
                    for (int j = 0; j < GT; ++j) s[j] = fma2(q[j][2 * c + 1], k[1], c == 0 ? mul2(q[j][0], k[0]) : fma2(q[j][2 * c], k[0], s[j]));
                }
#pragma unroll
                for (int j = 0; j < GT; ++j) {
                    const float2 y = of_pair(s[j]);
                    x[i][j] = y.x + y.y;
                }
            }
            // over the slices: entries by the lane's two lowest bits, heads by the next two
#pragma unroll
            for (int j = 0; j < GT; ++j) x[0][j] = xor_sum(x[0][j], x[1][j], 1), x[2][j] = xor_sum(x[2][j], x[3][j], 1);
#pragma unroll
            for (int j = 0; j < GT; ++j) x[0][j] = xor_sum(x[0][j], x[2][j], 2);
            float s[HPL];
            if constexpr (GT == 8) {
                x[0][0] = xor_sum(x[0][0], x[0][2], 4), x[0][1] = xor_sum(x[0][1], x[0][3], 4);
                x[0][4] = xor_sum(x[0][4], x[0][6], 4), x[0][5] = xor_sum(x[0][5], x[0][7], 4);
                s[0] = xor_sum(x[0][0], x[0][4], 8), s[HPL - 1] = xor_sum(x[0][1], x[0][5], 8);
            } else if constexpr (GT == 4) {
                x[0][0] = xor_sum(x[0][0], x[0][1], 4), x[0][2] = xor_sum(x[0][2], x[0][3], 4);
                s[0] = xor_sum(x[0][0], x[0][2], 8);
            } else {
                x[0][0] = xor_sum(x[0][0], x[0][1], 4);
                s[0] = xor_sum(x[0][0], x[0][0], 8);
            }
            const uint32_t mine = half * 4u + turn, e = base + mine, h0 = head_of(0);  // this lane's entry, its first head
            const bool any_bad = __any_sync(0xffffffffu, bad);
            if (e < at.t0 || e >= at.t1 || (any_bad && paged_page(a.c, list.slot[at.row], e) == PAGED_NONE)) {
#pragma unroll
                for (int h = 0; h < HPL; ++h) s[h] = -INFINITY;
            }
            float corr[HPL], p[HPL];
            bool moved = false;
#pragma unroll
            for (int h = 0; h < HPL; ++h) {
                if (a.scores && h0 + h < G && e >= at.t0 && e < at.t1)
                    a.scores[((size_t)(a.row0 + at.row) * a.q_heads + head0 + h0 + h) * a.ld_scores + e] = s[h];
                float mx = s[h];
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float m_new = fmaxf(m_run[h], mx), use = m_new == -INFINITY ? 0.0f : m_new;
                moved |= m_new > m_run[h];
                corr[h] = fast_exp2(m_run[h] - use);
                p[h] = fast_exp2(s[h] - use);
                l_run[h] = l_run[h] * corr[h] + p[h];  // this lane's entries
                m_run[h] = m_new;
            }
            if constexpr (HPL == 2)
                *reinterpret_cast<float4*>(s_p + mine * GT + h0) = make_float4(p[0], p[0], p[1], p[1]);
            else
                s_p[mine * GT + h0] = make_float2(p[0], p[0]);
            const bool rescale = __any_sync(0xffffffffu, moved);
            if (rescale && turn == 0 && half == 0) {
#pragma unroll
                for (int h = 0; h < HPL; ++h) s_corr[h0 + h] = corr[h];
            }
            __syncwarp();
            if (rescale) {
#pragma unroll
                for (int j = 0; j < GT; ++j) {
                    const float c = s_corr[j];
                    const uint64_t cc = pair_of(c, c);
#pragma unroll
                    for (int i = 0; i < 2 * DV; ++i) acc[j][i] = mul2(acc[j][i], cc);
                }
            }
#pragma unroll
            for (uint32_t t = 0; t < LANES_TILE; ++t) {
                uint64_t w[GT];
#pragma unroll
                for (int j = 0; j < GT; j += 2) {
                    const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(s_p + t * GT + j);
                    w[j] = y.x, w[j + 1] = y.y;
                }
#pragma unroll
                for (uint32_t i = 0; i < DV; ++i) {
                    const uint32_t d = (lane + 32u * i) * 4u;
                    uint64_t v[2] = {0u, 0u};
                    if (d < hd) load4(tV + t * hd + d, v);
#pragma unroll
                    for (int j = 0; j < GT; ++j) acc[j][2 * i] = fma2(w[j], v[0], acc[j][2 * i]), acc[j][2 * i + 1] = fma2(w[j], v[1], acc[j][2 * i + 1]);
                }
            }
            __syncwarp();  // the weights have been read
        }
        if (at.tile + 1u == at.tiles || f + 1u == count) {  // this warp's part of the unit
            const size_t part = (((size_t)at.row * units + at.unit + worker) * warps + warp) * a.heads_at_once;
            const uint32_t h0 = head_of(0);
#pragma unroll
            for (int h = 0; h < HPL; ++h) {
                float l = l_run[h];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (turn == 0 && half == 0 && h0 + h < G) a.part_m[part + h0 + h] = m_run[h], a.part_l[part + h0 + h] = l;
            }
#pragma unroll
            for (uint32_t j = 0; j < GT; ++j)
                if (j < G)
#pragma unroll
                    for (uint32_t i = 0; i < DV; ++i) {
                        const uint32_t d = (lane + 32u * i) * 4u;
                        if (d >= hd) continue;
                        const float2 y = of_pair(acc[j][2 * i]), z = of_pair(acc[j][2 * i + 1]);
                        *reinterpret_cast<float4*>(a.part_o + (part + j) * hd + d) = make_float4(y.x, y.y, z.x, z.y);
                    }
        }
        entering = paged_list_next(list, at, rows, units, span);
    }
    cp_async_wait<0>();
    if (bad) atomicOr(a.status, 1u);
}

uint32_t lanes_smem(uint32_t warps, uint32_t gt, uint32_t rb) {
    return lanes_rings(warps, gt) + warps * (LANES_STAGES * 2u * LANES_TILE * rb);
}
uint32_t lanes_gt(uint32_t heads) { return heads > 4u ? 8u : (heads > 2u ? 4u : 2u); }

template <typename ET, int GT, int DQ>
cudaError_t launch(M40llmCudaContext* ctx, const PagedAttnArgs& a, const PagedLanes& l) {
    const uint32_t smem = lanes_smem(l.warps, GT, a.c.hd * (uint32_t)sizeof(ET));
    const cudaError_t e = cudaFuncSetAttribute(paged_lanes_kernel<ET, GT, DQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PAGED_SMEM_MOST);
    if (e != cudaSuccess) return e;
    return m40_launch_dependent(paged_lanes_kernel<ET, GT, DQ>, dim3(a.workers), dim3(l.warps * 32u), smem, ctx->decode_stream, a);
}
template <typename ET>
cudaError_t launch_size(M40llmCudaContext* ctx, const PagedAttnArgs& a, const PagedLanes& l) {
    const uint32_t gt = lanes_gt(l.heads_at_once);
    if (a.c.hd <= 128u) return gt == 8u ? launch<ET, 8, 2>(ctx, a, l) : (gt == 4u ? launch<ET, 4, 2>(ctx, a, l) : launch<ET, 2, 2>(ctx, a, l));
    if (a.c.hd <= 256u) return gt == 4u ? launch<ET, 4, 4>(ctx, a, l) : launch<ET, 2, 4>(ctx, a, l);
    return launch<ET, 2, 8>(ctx, a, l);
}

}  // namespace

bool m40_paged_lanes(const M40llmCudaContext* ctx, const M40llmPagedCache* cache, uint32_t group, PagedLanes* out) {
    const uint32_t rb = cache->head_dim * (cache->elem_dtype == M40LLM_DT_F32 ? 4u : 2u);
    if (!m40_paged_vec16(cache)) return false;
    // what the registers hold of queries and outputs: 8 heads of 128 dimensions
    const uint32_t most = cache->head_dim <= 128u ? 8u : (cache->head_dim <= 256u ? 4u : 2u), shares = (group + most - 1u) / most;
    out->heads_at_once = (group + shares - 1u) / shares;
    // Rings of up to 100 KB and two CTAs on an SM, so that the next launch's CTAs find room as these end: 9 rows of up to 4097 f32 entries 20.0 us, with one CTA of
    // twice the warps 20.9, one row of 64 entries 7.7 against 9.0.
    out->warps = rb <= 512u ? 4u : (rb <= 1024u ? 2u : 1u);
    out->ctas = paged_list_ctas((uint32_t)ctx->sm_count, 2u, out->warps);
    return true;
}

cudaError_t m40_paged_lanes_launch(M40llmCudaContext* ctx, const PagedAttnArgs& a, const PagedLanes& l, bool f32) {
    return f32 ? launch_size<float>(ctx, a, l) : launch_size<__half>(ctx, a, l);
}
