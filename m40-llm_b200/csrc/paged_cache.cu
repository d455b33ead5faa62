// A key / value cache in pages: append (with rotation) and eviction by accumulated attention weight.
#include "paged.cuh"
#include "stack_math.cuh"

namespace {

// ------------------------------------------------------------------------------------------------------------------ append
struct AppendArgs {
    PagedView c;
    const float* q;
    const float* k;
    const float* v;
    float* q_out;
    const double* turns;
    const uint32_t* row_slot;
    const uint32_t* row_entry;
    const uint32_t* row_pos;
    uint32_t* entry_pos;
    float* weights;
    uint32_t* status;
    uint32_t q_heads, pairs, layout, ld_q, ld_k, ld_entry;
};

// CTA = (row, share of the row's heads). The row's rotation table is made once per CTA; the whole turns are dropped in double, where
// pos * turns is exact enough for any position, so that the single-precision sine and cosine see at most half a turn.
// Thread = one pair of one head (what lies behind the rotated part goes in pairs of neighbours). Bound by the launch for a step's
// rows and by the bytes of q, k and v for prompts.
template <typename ET>
__global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs a) {
    extern __shared__ float2 cs[];  // [pairs] cosine, sine
    pdl_wait();
    pdl_trigger();
    const uint32_t row = blockIdx.x, tid = threadIdx.x, hd = a.c.hd, half = (hd + 1u) / 2u;
    const uint32_t slot = a.row_slot[row], e = a.row_entry[row], pos = a.row_pos ? a.row_pos[row] : 0u;
    const bool inside = slot < a.c.slots && e < paged_capacity(a.c);
    const uint32_t page = inside ? paged_page(a.c, slot, e) : PAGED_NONE;
    for (uint32_t i = tid; i < a.pairs; i += blockDim.x) {
        const double t = (double)pos * a.turns[i];
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        cs[i] = make_float2(c, s);
    }
    __syncthreads();
    if (page == PAGED_NONE && tid == 0 && blockIdx.y == 0) atomicOr(a.status, 2u);
    const uint32_t heads = a.q_heads + 2u * a.c.kv_heads;
    for (uint32_t u = blockIdx.y * blockDim.x + tid; u < heads * half; u += gridDim.y * blockDim.x) {
        uint32_t head = u / half;
        const uint32_t j = u - head * half;
        const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.c.kv_heads, turn = j < a.pairs && !is_v;
        if (!is_q) head -= is_v ? a.q_heads + a.c.kv_heads : a.q_heads;
        uint32_t i0 = 2u * j, i1 = 2u * j + 1u;
        if (a.layout == 1u) {  // pairs (j, j + pairs), what is left behind them; values go alike, for whole lines
            if (j < a.pairs) i0 = j, i1 = j + a.pairs;
        }
        const float* src = (is_q ? a.q + (size_t)row * a.ld_q : (is_v ? a.v : a.k) + (size_t)row * a.ld_k) + (size_t)head * hd;
        float x = src[i0], y = i1 < hd ? src[i1] : 0.0f;
        if (turn) {
            const float2 t = cs[j];
            const float rx = x * t.x - y * t.y, ry = x * t.y + y * t.x;
            x = rx, y = ry;
        }
        if (is_q) {
            float* dst = a.q_out + ((size_t)row * a.q_heads + head) * hd;
            dst[i0] = x;
            if (i1 < hd) dst[i1] = y;
        } else if (page != PAGED_NONE) {
            ET* dst = reinterpret_cast<ET*>(is_v ? a.c.v : a.c.k) + paged_row(a.c, page, head, e);
            m40_store_elem(dst + i0, x);
            if (i1 < hd) m40_store_elem(dst + i1, y);
        }
    }
    if (page != PAGED_NONE && blockIdx.y == 0)
        for (uint32_t h = tid; h < a.c.kv_heads; h += blockDim.x) {
            const size_t at = ((size_t)slot * a.c.kv_heads + h) * a.ld_entry + e;
            if (a.entry_pos) a.entry_pos[at] = pos;
            if (a.weights) a.weights[at] = 0.0f;
        }
}

// ---------------------------------------------------------------------------------------------------------------- eviction
struct EvictArgs {
    PagedView c, to;
    const uint32_t* seq;
    const uint32_t* len;
    const float* weights;
    float* weights_out;
    const uint32_t* entry_pos;
    uint32_t* entry_pos_out;
    uint32_t* origin;   // [count][kv_heads][keep]
    uint32_t* new_len;  // [count]
    uint32_t* holes;    // scratch [count][kv_heads][keep]: free places below the new end
    uint32_t* late;     // scratch, likewise: kept entries behind it
    uint32_t* status;
    uint32_t keep, first, recent, ld, bound, in_place;
};

constexpr uint32_t SELECT_THREADS = 1024;

// Larger is better. Held entries come before every weight (+inf is 0xff800000), NaN after every other.
__device__ __forceinline__ uint32_t evict_key(float w, bool held) {
    if (held) return 0xffffffffu;
    if (isnan(w)) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);  // -0 is 0
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// Sum of x over the threads before this one; `total` gets the block's. Two barriers.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* warps, uint32_t* total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t v = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    __syncthreads();
    if (lane == 31u) warps[warp] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t w = 0; w < SELECT_THREADS / 32; ++w) {
        if (w < warp) before += warps[w];
        all += warps[w];
    }
    *total = all;
    return before + v - x;
}

// CTA = (listed sequence, kv head). The key of the last kept entry is found by its bytes, from the highest down (256 bins each); one more pass over
// the entries in order deals the ties, and notes the holes below the new end and the kept entries behind it.
__global__ void __launch_bounds__(SELECT_THREADS) evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t bins[256], warps[SELECT_THREADS / 32], s_pick[2], s_end;
    pdl_wait();
    pdl_trigger();
    const uint32_t i = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
    const uint32_t slot = a.seq[i], len = a.len[i];
    bool bad = slot >= a.c.slots || len > a.bound;
    if (tid == 0) s_end = 0u;
    int twice = 0;
    for (uint32_t j = tid; j < i; j += SELECT_THREADS) twice |= a.seq[j] == slot;
    if (__syncthreads_or(twice)) bad = true;
    uint32_t* from = a.origin + ((size_t)i * a.c.kv_heads + h) * a.keep;
    const uint32_t kept = bad ? 0u : min(len, a.keep);
    if (tid == 0 && h == 0) {
        a.new_len[i] = kept;
        if (bad) atomicOr(a.status, 1u);
    }
    for (uint32_t e = kept + tid; e < a.keep; e += SELECT_THREADS) from[e] = PAGED_NONE;
    if (kept == 0 || len <= a.keep) {
        for (uint32_t e = tid; e < kept; e += SELECT_THREADS) from[e] = e;
        return;
    }
    const size_t base = ((size_t)slot * a.c.kv_heads + h) * a.ld;
    const float* w = a.weights + base;
    const uint32_t* pos = a.entry_pos ? a.entry_pos + base : nullptr;
    uint32_t newest = 0;
    if (pos)
        for (uint32_t e = tid; e < len; e += SELECT_THREADS) newest = max(newest, pos[e]);
    else
        newest = len - 1u;
    newest = __reduce_max_sync(0xffffffffu, newest);
    if ((tid & 31u) == 0) atomicMax(&s_end, newest);
    __syncthreads();
    newest = s_end;
    auto key = [&](uint32_t e) {
        const uint32_t p = pos ? pos[e] : e;
        return evict_key(w[e], p < a.first || newest - p < a.recent);
    };
    uint32_t prefix = 0, want = a.keep;  // the want-th largest among the keys that begin with prefix
    for (int byte = 3; byte >= 0; --byte) {
        const uint32_t high = byte == 3 ? 0u : 0xffffffffu << (8 * (byte + 1));
        for (uint32_t b = tid; b < 256u; b += SELECT_THREADS) bins[b] = 0;
        __syncthreads();
        for (uint32_t e = tid; e < len; e += SELECT_THREADS) {
            const uint32_t k = key(e);
            if ((k & high) == prefix) atomicAdd(&bins[(k >> (8 * byte)) & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t b = 255u, above = 0;
            while (above + bins[b] < want) above += bins[b--];
            s_pick[0] = b;
            s_pick[1] = want - above;
        }
        __syncthreads();
        prefix |= s_pick[0] << (8 * byte);
        want = s_pick[1];
        __syncthreads();
    }
    uint32_t* holes = a.holes + ((size_t)i * a.c.kv_heads + h) * a.keep;
    uint32_t* late = a.late + ((size_t)i * a.c.kv_heads + h) * a.keep;
    uint32_t ties = 0, n_holes = 0, n_late = 0;
    for (uint32_t e0 = 0; e0 < len; e0 += SELECT_THREADS) {
        const uint32_t e = e0 + tid;
        const uint32_t k = e < len ? key(e) : 0u;
        const bool tie = e < len && k == prefix;
        uint32_t total;
        const uint32_t rank = ties + block_scan(tie ? 1u : 0u, warps, &total);
        ties += total;
        const bool stays = e < len && (k > prefix || (tie && rank < want));
        const bool hole = e < a.keep && !stays, behind = e >= a.keep && stays;
        const uint32_t nh = n_holes + block_scan(hole ? 1u : 0u, warps, &total);
        n_holes += total;
        const uint32_t nl = n_late + block_scan(behind ? 1u : 0u, warps, &total);
        n_late += total;
        if (stays && e < a.keep) from[e] = e;
        if (hole) holes[nh] = e;
        if (behind) late[nl] = e;
    }
    __syncthreads();
    for (uint32_t j = tid; j < n_holes; j += SELECT_THREADS) from[holes[j]] = late[j];
}

// Warp = one kept place of one kv head. In place a source lies behind the new end and a target before it, so that no copy reads what
// another writes.
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a, uint32_t row_bytes, uint32_t elem, uint32_t vec) {
    pdl_wait();
    pdl_trigger();
    const uint32_t i = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31u, place = blockIdx.x * 8u + (threadIdx.x >> 5);
    if (place >= a.keep) return;
    const uint32_t src = a.origin[((size_t)i * a.c.kv_heads + h) * a.keep + place];
    if (src == PAGED_NONE) return;
    const uint32_t slot = a.seq[i];
    const size_t base = ((size_t)slot * a.c.kv_heads + h) * a.ld;
    if (lane == 0) {
        if (a.weights_out && (src != place || a.weights_out != a.weights)) a.weights_out[base + place] = a.weights[base + src];
        if (a.entry_pos_out && (src != place || a.entry_pos_out != a.entry_pos)) a.entry_pos_out[base + place] = a.entry_pos ? a.entry_pos[base + src] : src;
    }
    if (a.in_place && src == place) return;
    const uint32_t from = paged_page(a.c, slot, src), into = paged_page(a.to, slot, place);
    if (from == PAGED_NONE || into == PAGED_NONE) {
        if (lane == 0) atomicOr(a.status, from == PAGED_NONE ? 1u : 2u);
        return;
    }
    const size_t s = paged_row(a.c, from, h, src) * elem, d = paged_row(a.to, into, h, place) * elem;
    if (vec) {
        for (uint32_t b = lane * 16u; b < row_bytes; b += 512u) {
            const uint4 x = *reinterpret_cast<const uint4*>(a.c.k + s + b), y = *reinterpret_cast<const uint4*>(a.c.v + s + b);
            *reinterpret_cast<uint4*>(a.to.k + d + b) = x;
            *reinterpret_cast<uint4*>(a.to.v + d + b) = y;
        }
    } else {
        for (uint32_t b = lane * 2u; b < row_bytes; b += 64u) {
            *reinterpret_cast<uint16_t*>(a.to.k + d + b) = *reinterpret_cast<const uint16_t*>(a.c.k + s + b);
            *reinterpret_cast<uint16_t*>(a.to.v + d + b) = *reinterpret_cast<const uint16_t*>(a.c.v + s + b);
        }
    }
}

}  // namespace

extern "C" {

int m40llm_paged_append_async(M40llmCudaContext* ctx, const M40llmPagedCache* cache, const M40llmPagedAppend* c) {
    if (!ctx || !cache || !c || !c->k || !c->v || !c->row_slot || !c->row_entry) return -1;
    AppendArgs a = {};
    int rc = m40_paged_view(cache, &a.c);
    if (rc != 0) return rc;
    if (c->rows == 0) return -2;
    if (c->q_heads && (!c->q || !c->q_out)) return -1;
    if (((c->pairs || c->entry_pos) && !c->row_pos) || (c->pairs && !c->turns)) return -1;
    const uint64_t wide = (uint64_t)c->q_heads * cache->head_dim, tight = (uint64_t)cache->kv_heads * cache->head_dim;
    if (wide > 0xffffffffull || tight > 0xffffffffull || 2ull * c->pairs > cache->head_dim || c->rope_layout > 1u) return -2;
    if (c->ld && (c->ld < wide || c->ld < tight)) return -2;
    if ((c->entry_pos || c->weights) && c->ld_entry < paged_capacity(a.c)) return -2;
    if (m40_ensure_device(ctx) != 0) return -1;
    a.q = (const float*)c->q;
    a.k = (const float*)c->k;
    a.v = (const float*)c->v;
    a.q_out = (float*)c->q_out;
    a.turns = (const double*)c->turns;
    a.row_slot = c->row_slot;
    a.row_entry = c->row_entry;
    a.row_pos = c->row_pos;
    a.entry_pos = c->entry_pos;
    a.weights = (float*)c->weights;
    a.status = ctx->d_status;
    a.q_heads = c->q_heads;
    a.pairs = c->pairs;
    a.layout = c->rope_layout;
    a.ld_q = c->ld ? c->ld : (uint32_t)wide;
    a.ld_k = c->ld ? c->ld : (uint32_t)tight;
    a.ld_entry = c->ld_entry;
    const uint64_t units = ((uint64_t)c->q_heads + 2ull * cache->kv_heads) * ((cache->head_dim + 1u) / 2u);
    if (units > 0x7fffffffull) return M40LLM_ERR_LIMIT;
    const uint32_t most = (uint32_t)((units + 255u) / 256u), want = (uint32_t)(4 * ctx->sm_count) / c->rows;
    const dim3 grid(c->rows, want < 1u ? 1u : (want < most ? want : most));
    const size_t smem = (size_t)c->pairs * sizeof(float2);
    const cudaError_t e = cache->elem_dtype == M40LLM_DT_F32
                              ? m40_launch_dependent(paged_append_kernel<float>, grid, dim3(256), smem, ctx->decode_stream, a)
                              : m40_launch_dependent(paged_append_kernel<__half>, grid, dim3(256), smem, ctx->decode_stream, a);
    M40_COUNT_LAUNCH(ctx);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int m40llm_paged_evict_async(M40llmCudaContext* ctx, const M40llmPagedCache* cache, const M40llmPagedEvict* c) {
    if (!ctx || !cache || !c || !c->seq || !c->len || !c->weights || !c->new_len) return -1;
    EvictArgs a = {};
    int rc = m40_paged_view(cache, &a.c);
    if (rc != 0) return rc;
    const M40llmPagedCache* to = c->to ? c->to : cache;
    rc = m40_paged_view(to, &a.to);
    if (rc != 0) return rc;
    const uint32_t capacity = paged_capacity(a.c);
    if (c->count == 0 || c->keep == 0 || c->keep > capacity || c->keep > paged_capacity(a.to)) return -2;
    if ((uint64_t)c->first + c->recent > c->keep || c->ld < capacity || c->max_len > capacity) return -2;
    if (to->kv_heads != cache->kv_heads || to->head_dim != cache->head_dim || to->slots < cache->slots) return -2;
    if (to->elem_dtype != cache->elem_dtype) return -4;
    if (c->count > 65535u) return M40LLM_ERR_LIMIT;
    if (m40_ensure_device(ctx) != 0) return -1;
    // the same pool through the same table is the cache itself
    a.in_place = to->k == cache->k && to->v == cache->v && to->table == cache->table ? 1u : 0u;
    a.seq = c->seq;
    a.len = c->len;
    a.weights = (const float*)c->weights;
    a.weights_out = (float*)c->weights_out;
    a.entry_pos = c->entry_pos;
    a.entry_pos_out = c->entry_pos_out;
    a.new_len = c->new_len;
    a.status = ctx->d_status;
    a.keep = c->keep;
    a.first = c->first;
    a.recent = c->recent;
    a.ld = c->ld;
    a.bound = c->max_len ? c->max_len : capacity;
    const size_t places = (size_t)c->count * cache->kv_heads * c->keep;
    uint32_t* work = (uint32_t*)m40_ensure_scratch(ctx, 1, 3 * places * sizeof(uint32_t), 0);
    if (!work) return -5;
    a.holes = work;
    a.late = work + places;
    a.origin = c->origin ? c->origin : work + 2 * places;
    cudaError_t e = m40_launch_dependent(evict_select_kernel, dim3(cache->kv_heads, c->count), dim3(SELECT_THREADS), 0, ctx->decode_stream, a);
    M40_COUNT_LAUNCH(ctx);
    if (e != cudaSuccess) return -3;
    const uint32_t elem = cache->elem_dtype == M40LLM_DT_F32 ? 4u : 2u;
    e = m40_launch_dependent(evict_move_kernel, dim3((c->keep + 7u) / 8u, cache->kv_heads, c->count), dim3(256), 0, ctx->decode_stream, a,
                             cache->head_dim * elem, elem, m40_paged_vec16(cache) && m40_paged_vec16(to) ? 1u : 0u);
    M40_COUNT_LAUNCH(ctx);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // extern "C"
