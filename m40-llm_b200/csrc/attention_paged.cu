// Attention of single tokens over a cache in pages: m40llm_attention_paged_async.
//
// Work is dealt as (row, kv head, chunk of entries): softmax statistics are kept with a running maximum in base 2, and the chunks'
// (maximum, sum, unnormalised output) meet in paged_merge_kernel in a fixed order. Where accumulated weights are asked for, the
// scores are kept in scratch and paged_weights_kernel turns them into weights once the maximum and sum of every row are known.
//   paged_rows_kernel   any head size, group size and type: f32 multiply-adds on tiles in shared memory
#include "attention_mma.cuh"
#include "paged.cuh"
#include "stack_math.cuh"

namespace {

using namespace attn_mma;

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
    uint32_t rows, q_heads, group, splits, chunk, bound, ld_weights, ld_scores;
    float scale;  // times log2(e)
};

// The entries [begin, end) of a row; false for a row outside the cache.
__device__ __forceinline__ bool paged_row_range(const PagedAttnArgs& a, uint32_t row, uint32_t* slot, uint32_t* begin, uint32_t* end) {
    *slot = a.row_slot[row];
    *end = a.row_len[row];
    *begin = a.row_begin ? a.row_begin[row] : 0u;
    return *slot < a.c.slots && *end <= a.bound;
}
// The part of them that split s covers; chunks are counted from the tile that `begin` lies in.
__device__ __forceinline__ void paged_chunk(const PagedAttnArgs& a, uint32_t split, uint32_t begin, uint32_t end, uint32_t* t0, uint32_t* t1) {
    const uint64_t lo = (uint64_t)(begin & ~63u) + (uint64_t)split * a.chunk, hi = lo + a.chunk;
    *t0 = lo > begin ? (lo < end ? (uint32_t)lo : end) : begin;
    *t1 = hi < end ? (uint32_t)hi : end;
    if (*t1 < *t0) *t1 = *t0;
}

constexpr uint32_t ROWS_THREADS = 128;

// CTA = (row, GT q heads of one kv head, chunk). Tiles of T entries of keys and values in shared memory, two in flight. Scores: thread =
// (entry, slice of the dimensions), the slices meet in shared memory; softmax: warp = head, lane = entry; output: thread = dimensions.
template <typename ET, int GT, int DV>
__global__ void __launch_bounds__(ROWS_THREADS) paged_rows_kernel(PagedAttnArgs a, uint32_t T, uint32_t vec, uint32_t pitch) {
    extern __shared__ __align__(16) unsigned char smem[];
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

// CTA = (q head, row): the chunks' parts in order.
__global__ void __launch_bounds__(128) paged_merge_kernel(PagedAttnArgs a) {
    __shared__ float red[8];
    pdl_wait();
    pdl_trigger();
    const uint32_t tid = threadIdx.x, hd = a.c.hd;
    const size_t head = (size_t)blockIdx.y * a.q_heads + blockIdx.x, base = head * a.splits;
    float M = -INFINITY, nan = 0.0f;
    for (uint32_t s = tid; s < a.splits; s += 128u) {
        const float l = a.part_l[base + s];
        if (l != 0.0f) M = fmaxf(M, a.part_m[base + s]);
        if (isnan(l)) nan = 1.0f;
    }
    M = warp_max(M);
    nan = warp_max(nan);
    if ((tid & 31u) == 0) red[tid >> 5] = M, red[4 + (tid >> 5)] = nan;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float L = 0.0f;
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float l = a.part_l[base + s];
        if (l != 0.0f) L += l * exp2f(a.part_m[base + s] - M);
    }
    const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : NAN);
    for (uint32_t d = tid; d < hd; d += 128u) {
        float o = 0.0f;
        for (uint32_t s = 0; s < a.splits; ++s) {
            const float l = a.part_l[base + s];
            if (l != 0.0f) o = fmaf(exp2f(a.part_m[base + s] - M), a.part_o[(base + s) * hd + d], o);
        }
        a.out[head * hd + d] = L == 0.0f ? 0.0f : o * inv;
    }
    if (a.stat && tid == 0) a.stat[2 * head] = M, a.stat[2 * head + 1] = inv;
}

// CTA = (256 entries, kv head, row); only the first row of a slot works, for all rows of the slot in their order, so that sums do not
// depend on who comes first.
__global__ void __launch_bounds__(256) paged_weights_kernel(PagedAttnArgs a) {
    pdl_wait();
    pdl_trigger();
    const uint32_t row = blockIdx.z, h = blockIdx.y, e = blockIdx.x * 256u + threadIdx.x;
    const uint32_t slot = a.row_slot[row];
    if (slot >= a.c.slots) return;
    uint32_t most = 0, skip = 0;
    for (uint32_t r = 0; r < a.rows; ++r) {
        uint32_t s, b, n;
        const bool inside = paged_row_range(a, r, &s, &b, &n);
        if (s != slot) continue;
        if (r < row || !inside) skip = 1;
        most = max(most, n);
    }
    if (skip || e >= most) return;
    const size_t at = ((size_t)slot * a.c.kv_heads + h) * a.ld_weights + e;
    float w = a.weights_in ? a.weights_in[at] : 0.0f;
    for (uint32_t r = row; r < a.rows; ++r) {
        uint32_t s, b, n;
        paged_row_range(a, r, &s, &b, &n);
        if (s != slot || e < b || e >= n) continue;
        float sum = 0.0f;
        for (uint32_t g = 0; g < a.group; ++g) {
            const size_t head = (size_t)r * a.q_heads + h * a.group + g;
            sum += exp2f(a.scores[head * a.ld_scores + e] - a.stat[2 * head]) * a.stat[2 * head + 1];
        }
        w += sum;
    }
    a.weights_out[at] = w;
}

template <typename ET, int GT>
cudaError_t launch_rows(const PagedAttnArgs& a, dim3 grid, uint32_t T, uint32_t vec, uint32_t pitch, size_t smem, cudaStream_t s) {
    const uint32_t dv = (a.c.hd + ROWS_THREADS - 1) / ROWS_THREADS;
    void (*kernel)(PagedAttnArgs, uint32_t, uint32_t, uint32_t) =
        dv == 1 ? paged_rows_kernel<ET, GT, 1> : (dv == 2 ? paged_rows_kernel<ET, GT, 2> : paged_rows_kernel<ET, GT, 4>);
    if (smem > 48u * 1024u) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
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
    if (c->rows > 65535u || c->q_heads > 65535u) return M40LLM_ERR_LIMIT;
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
    a.bound = c->max_len ? c->max_len : capacity;
    a.scale = c->scale * LOG2E;
    const uint32_t covered = a.bound;
    const uint64_t work = (uint64_t)c->rows * cache->kv_heads * covered, target = 2ull * (uint64_t)ctx->sm_count;
    uint64_t chunk = (work + target - 1) / target;
    chunk = chunk < 128u ? 128u : (chunk > 1024u ? 1024u : chunk);
    chunk = (chunk + 63u) & ~63ull;
    if ((covered + chunk - 1) / chunk > 256u) chunk = ((covered + 255u) / 256u + 63u) & ~63ull;
    a.chunk = (uint32_t)chunk;
    a.splits = (uint32_t)((covered + chunk - 1) / chunk);
    const size_t heads = (size_t)c->rows * c->q_heads;
    if (a.splits > 1 || c->weights_out) {
        a.ld_scores = c->weights_out ? a.bound : 0u;
        const size_t parts = heads * a.splits, floats = parts * (hd + 2) + heads * 2 + heads * (size_t)a.ld_scores;
        float* work_area = (float*)m40_ensure_scratch(ctx, 1, floats * sizeof(float), 0);
        if (!work_area) return -5;
        a.part_o = work_area;
        a.part_m = a.part_o + parts * hd;
        a.part_l = a.part_m + parts;
        if (c->weights_out) {
            a.stat = a.part_l + parts;
            a.scores = a.stat + 2 * heads;
        }
    }
    cudaStream_t s = ctx->decode_stream;
    const bool f32 = cache->elem_dtype == M40LLM_DT_F32;
    const uint32_t elem = f32 ? 4u : 2u, hd4 = (hd + 3u) & ~3u;
    const uint32_t T = hd4 * elem > 1024u ? 16u : 32u, pitch = ((hd4 * elem + 15u) & ~15u) / elem + 16u / elem;
    const uint32_t vec = m40_paged_vec16(cache) ? 1u : 0u;
    const uint32_t gt = a.group >= 8u ? 8u : (a.group >= 4u ? 4u : (a.group >= 2u ? 2u : 1u)), subgroups = (a.group + gt - 1) / gt;
    const dim3 grid(a.splits, cache->kv_heads * subgroups, c->rows);
    if (grid.y > 65535u) return M40LLM_ERR_LIMIT;
    const size_t smem = ((size_t)gt * hd4 + ROWS_THREADS * gt + gt * 32u + 8u + 64u) * 4u + 4ull * T * pitch * elem;
    cudaError_t e;
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
    if (e != cudaSuccess) return cudaGetLastError(), -3;
    if (a.splits > 1 || a.scores) {
        e = m40_launch_dependent(paged_merge_kernel, dim3(c->q_heads, c->rows), dim3(128), 0, s, a);
        M40_COUNT_LAUNCH(ctx);
    }
    if (e == cudaSuccess && a.scores) {
        e = m40_launch_dependent(paged_weights_kernel, dim3((a.bound + 255u) / 256u, cache->kv_heads, c->rows), dim3(256), 0, s, a);
        M40_COUNT_LAUNCH(ctx);
    }
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -3;
}
