// A key / value cache in pages: append (with rotation) and eviction by accumulated attention weight.
#include "paged.cuh"
#include "stack_math.cuh"
#include "tc_ptx.cuh"

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

__device__ __forceinline__ void store4(float* p, const float4& v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__half* p, const float4& v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// The same for heads of eights and 16-byte aligned rows. Thread = units of eight values of a head: four pairs, or eight values that do not turn. Its loads go
// out before the row's table is made: one after the other they took 17.4 us for 2001 rows of 20 heads of 128 (2.5 units a thread), now 9.7. What is beyond three units
// goes one by one, beside the other CTAs' loads: 48 heads of 128 (6 units) 18.4 us against a floor of 14.0, 12 heads 5.3 against 3.5.
constexpr uint32_t APPEND_THREADS = 128, APPEND_UNITS = 3;
template <typename ET>
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_vec_kernel(AppendArgs a) {
    extern __shared__ float2 cs[];  // [pairs] cosine, sine
    pdl_wait();
    pdl_trigger();
    const uint32_t row = blockIdx.x, tid = threadIdx.x, hd = a.c.hd, each = hd / 8u, turning = a.pairs / 4u;
    const uint32_t units = (a.q_heads + 2u * a.c.kv_heads) * each, step = gridDim.y * APPEND_THREADS;
    struct Unit {
        const float* src;
        uint32_t head, i0, i1, j;
        bool is_q, is_v;
    };
    const auto unit_of = [&](uint32_t u) {
        Unit x;
        x.head = u / each;
        x.j = u - x.head * each;
        x.is_q = x.head < a.q_heads, x.is_v = x.head >= a.q_heads + a.c.kv_heads;
        if (!x.is_q) x.head -= x.is_v ? a.q_heads + a.c.kv_heads : a.q_heads;
        const bool halves = a.layout == 1u && x.j < turning;
        x.i0 = halves ? 4u * x.j : 8u * x.j, x.i1 = halves ? 4u * x.j + a.pairs : 8u * x.j + 4u;
        x.src = (x.is_q ? a.q + (size_t)row * a.ld_q : (x.is_v ? a.v : a.k) + (size_t)row * a.ld_k) + (size_t)x.head * hd;
        return x;
    };
    const uint32_t u0 = blockIdx.y * APPEND_THREADS + tid;
    float4 x[APPEND_UNITS], y[APPEND_UNITS];
#pragma unroll
    for (uint32_t k = 0; k < APPEND_UNITS; ++k)
        if (u0 + k * step < units) {
            const Unit n = unit_of(u0 + k * step);
            x[k] = *reinterpret_cast<const float4*>(n.src + n.i0), y[k] = *reinterpret_cast<const float4*>(n.src + n.i1);
        }
    const uint32_t slot = a.row_slot[row], e = a.row_entry[row], pos = a.row_pos ? a.row_pos[row] : 0u;
    const bool inside = slot < a.c.slots && e < paged_capacity(a.c);
    for (uint32_t i = tid; i < a.pairs; i += APPEND_THREADS) {
        const double t = (double)pos * a.turns[i];
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        cs[i] = make_float2(c, s);
    }
    const uint32_t page = inside ? paged_page(a.c, slot, e) : PAGED_NONE;
    __syncthreads();
    if (page == PAGED_NONE && tid == 0 && blockIdx.y == 0) atomicOr(a.status, 2u);
    const auto put = [&](const Unit& n, float4 p, float4 q) {
        if (n.j < turning && !n.is_v) {
            const float2 *t = cs + 4u * n.j, t0 = t[0], t1 = t[1], t2 = t[2], t3 = t[3];
            const float4 b = p, d = q;
            if (a.layout == 1u) {
                p = make_float4(b.x * t0.x - d.x * t0.y, b.y * t1.x - d.y * t1.y, b.z * t2.x - d.z * t2.y, b.w * t3.x - d.w * t3.y);
                q = make_float4(b.x * t0.y + d.x * t0.x, b.y * t1.y + d.y * t1.x, b.z * t2.y + d.z * t2.x, b.w * t3.y + d.w * t3.x);
            } else {
                p = make_float4(b.x * t0.x - b.y * t0.y, b.x * t0.y + b.y * t0.x, b.z * t1.x - b.w * t1.y, b.z * t1.y + b.w * t1.x);
                q = make_float4(d.x * t2.x - d.y * t2.y, d.x * t2.y + d.y * t2.x, d.z * t3.x - d.w * t3.y, d.z * t3.y + d.w * t3.x);
            }
        }
        if (n.is_q) {
            float* dst = a.q_out + ((size_t)row * a.q_heads + n.head) * hd;
            store4(dst + n.i0, p), store4(dst + n.i1, q);
        } else if (page != PAGED_NONE) {
            ET* dst = reinterpret_cast<ET*>(n.is_v ? a.c.v : a.c.k) + paged_row(a.c, page, n.head, e);
            store4(dst + n.i0, p), store4(dst + n.i1, q);
        }
    };
#pragma unroll
    for (uint32_t k = 0; k < APPEND_UNITS; ++k)
        if (u0 + k * step < units) put(unit_of(u0 + k * step), x[k], y[k]);
    for (uint32_t u = u0 + APPEND_UNITS * step; u < units; u += step) {
        const Unit n = unit_of(u);
        put(n, *reinterpret_cast<const float4*>(n.src + n.i0), *reinterpret_cast<const float4*>(n.src + n.i1));
    }
    if (page != PAGED_NONE && blockIdx.y == 0)
        for (uint32_t h = tid; h < a.c.kv_heads; h += APPEND_THREADS) {
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
    uint32_t* origin;   // [count][kv_heads][keep] or null
    uint32_t* new_len;  // [count]
    uint32_t* plan;     // scratch [count][kv_heads][keep]: a place's own entry, EVICT_HOLE + the hole's number, or PAGED_NONE beyond the new length
    uint32_t* late;     // scratch, likewise: kept entries behind the new end, in order
    uint32_t* kept;     // scratch [count]: the new lengths, which the copy gives out, as new_len may be the lengths that every CTA reads
    uint32_t* status;
    uint32_t keep, first, recent, ld, bound, in_place;
    uint32_t cached;    // entries that a CTA's shared memory holds
};

constexpr uint32_t SELECT_THREADS = 512, SELECT_WARPS = SELECT_THREADS / 32, EVICT_HOLE = 0x80000000u, SELECT_CLUSTER = 16;
constexpr uint32_t SELECT_CACHED = 24576;  // entries with key and position in 192 KB
constexpr int SELECT_BITS = 11, SELECT_BINS = 1 << SELECT_BITS, SELECT_GROUPS = SELECT_BINS / 32, SELECT_PASSES = 3;  // 32 bits in 11, 11 and 10
constexpr uint32_t SELECT_LIST = 2048;     // keys that every CTA sorts out by itself

// Larger is better. Held entries come before every weight (+inf is 0xff800000), NaN after every other.
__device__ __forceinline__ uint32_t evict_key(float w, bool held) {
    if (held) return 0xffffffffu;
    if (isnan(w)) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);  // -0 is 0
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// Sum over the warps before this one of a value per warp, and over all of them; `warps` is shared memory for SELECT_WARPS values. Two barriers.
__device__ __forceinline__ uint4 warps_before(const uint4& mine, uint4* warps, uint4* total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) warps[warp] = mine;
    __syncthreads();
    const uint4 x = lane < SELECT_WARPS ? warps[lane] : make_uint4(0, 0, 0, 0);
    const auto upto = [&](uint32_t v, uint32_t* all) {
        uint32_t sum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= (uint32_t)o) sum += u;
        }
        *all = __shfl_sync(0xffffffffu, sum, 31);
        return __shfl_sync(0xffffffffu, sum - v, warp);
    };
    uint4 r;
    r.x = upto(x.x, &total->x), r.y = upto(x.y, &total->y), r.z = upto(x.z, &total->z), r.w = upto(x.w, &total->w);
    return r;
}

struct SelectShared {
    uint32_t bins[SELECT_BINS];
    uint4 warps[SELECT_WARPS];
    uint32_t newest, found, pick[4];
    // what the CTAs of the cluster tell each other, by the teller's number
    uint32_t newest_of[SELECT_CLUSTER];
    uint32_t groups_of[SELECT_CLUSTER][SELECT_GROUPS];  // sums of 32 bins
    uint32_t bins_of[SELECT_CLUSTER][32];               // one group's bins
    uint4 counts_of[SELECT_CLUSTER];                    // larger and equal keys below the new end, then behind it
    uint32_t list[SELECT_LIST];                         // the keys of one bin, of all CTAs
};

// All threads of the cluster; what was stored into other CTAs' memory before it is there behind it.
__device__ __forceinline__ void cluster_meet() {
    __syncwarp();
    tc::cluster_sync_all();
}

// Sum over the lanes before this one.
__device__ __forceinline__ uint32_t lanes_before(uint32_t own) {
    uint32_t sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, sum, o);
        if ((threadIdx.x & 31u) >= (uint32_t)o) sum += u;
    }
    return sum - own;
}

// Cluster of CTAs = (listed sequence, kv head); a CTA has a run of its entries, their keys in shared memory where they fit (else they are made again in every
// pass). The key of the last kept entry is found by its bits from the highest down: a histogram of 11 bits per CTA, in groups of 32 bins; the groups' sums go to all
// CTAs, then the bins of the one group that matters, then, where these are at most 2048, the keys of the one bin that matters, which every CTA sorts
// out by itself (else two more histograms follow). Then the entries are counted once, larger and equal ones below and behind the new end, which gives every
// warp the numbers of its ties, holes and kept entries behind the end, so that the plan is written without an order of who comes first. What CTAs tell each other
// is stored into the others' memory before a barrier: loads from there took 400 cycles each. Against one CTA and four passes from memory: 4 x 8 heads
// of 8192 entries with the copy 76 -> 23.1 us, 8 heads of 32768 217 -> 27.1. Bound by the barriers of the cluster and a chain of short steps.
__global__ void __launch_bounds__(SELECT_THREADS) evict_select_kernel(EvictArgs a) {
    extern __shared__ __align__(16) uint32_t s_dyn[];  // [cached] keys, [cached] positions
    __shared__ SelectShared sh;
    uint32_t peers;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(peers));
    const uint32_t me = tc::cluster_rank(), h = blockIdx.x / peers, i = blockIdx.y, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (tid == 0) sh.newest = 0u, sh.found = 0u;
    pdl_wait();
    pdl_trigger();
    const uint32_t slot = a.seq[i], len = a.len[i];
    int twice = 0;
    for (uint32_t j = tid; j < i; j += SELECT_THREADS) twice |= a.seq[j] == slot;
    const bool bad = __syncthreads_or(twice) || slot >= a.c.slots || len > a.bound;  // the same in every CTA of the cluster
    uint32_t* plan = a.plan + ((size_t)i * a.c.kv_heads + h) * a.keep;
    const uint32_t kept = bad ? 0u : min(len, a.keep);
    if (tid == 0 && h == 0 && me == 0) {
        a.kept[i] = kept;
        if (bad) atomicOr(a.status, 1u);
    }
    const uint32_t all = me * SELECT_THREADS + tid, step = peers * SELECT_THREADS;
    for (uint32_t e = kept + all; e < a.keep; e += step) plan[e] = PAGED_NONE;
    if (kept == 0 || len <= a.keep) {
        for (uint32_t e = all; e < kept; e += step) plan[e] = e;
        return;
    }
    const size_t base = ((size_t)slot * a.c.kv_heads + h) * a.ld;
    const float* w = a.weights + base;
    const uint32_t* pos = a.entry_pos ? a.entry_pos + base : nullptr;
    // this CTA's entries [lo, hi), and in them the warp's [wlo, whi)
    const uint32_t per = (len + peers - 1u) / peers, lo = min(me * per, len), hi = min(lo + per, len), mine = hi - lo;
    const uint32_t per_warp = ((per + SELECT_WARPS - 1u) / SELECT_WARPS + 31u) & ~31u, wlo = min(lo + warp * per_warp, hi), whi = min(wlo + per_warp, hi);
    const bool cached = per <= a.cached;
    uint32_t* s_key = s_dyn;
    uint32_t* s_pos = s_dyn + a.cached;
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // every CTA of the cluster is there before anything is stored into it
    uint32_t newest = 0;
    if (pos) {
#pragma unroll 8
        for (uint32_t j = tid; j < mine; j += SELECT_THREADS) {
            const uint32_t p = pos[lo + j];
            if (cached) s_pos[j] = p, s_key[j] = evict_key(w[lo + j], false);
            newest = max(newest, p);
        }
        newest = __reduce_max_sync(0xffffffffu, newest);
        if (lane == 0) atomicMax(&sh.newest, newest);
        __syncthreads();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (tid < peers) tc::st_cluster(tc::map_to_rank(tc::smem_u32(&sh.newest_of[me]), tid), sh.newest);
        cluster_meet();
        newest = __reduce_max_sync(0xffffffffu, lane < peers ? sh.newest_of[lane] : 0u);
    } else {
        newest = len - 1u;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    const auto fresh = [&](uint32_t e) {
        const uint32_t p = pos ? pos[e] : e;
        return evict_key(w[e], p < a.first || newest - p < a.recent);
    };
    if (cached)
#pragma unroll 8
        for (uint32_t j = tid; j < mine; j += SELECT_THREADS) {
            if (!pos) {
                s_key[j] = fresh(lo + j);
            } else {
                const uint32_t p = s_pos[j];
                if (p < a.first || newest - p < a.recent) s_key[j] = 0xffffffffu;
            }
        }
    const auto key = [&](uint32_t e) { return cached ? s_key[e - lo] : fresh(e); };

    uint32_t prefix = 0, want = a.keep;  // the want-th largest among the keys that begin with prefix
#pragma unroll 1
    for (int pass = 0; pass < SELECT_PASSES; ++pass) {
        const int shift = pass == 0 ? 32 - SELECT_BITS : (pass == 1 ? 32 - 2 * SELECT_BITS : 0), bits = pass == 2 ? 32 - 2 * SELECT_BITS : SELECT_BITS;
        const uint32_t high = pass == 0 ? 0u : 0xffffffffu << (shift + bits);
        for (uint32_t b = tid; b < SELECT_BINS; b += SELECT_THREADS) sh.bins[b] = 0u;
        __syncthreads();
        // A warp whose keys are all in one bin (equal weights) adds once.
        for (uint32_t j0 = 0; j0 < mine; j0 += SELECT_THREADS) {
            const uint32_t j = j0 + tid, k = j < mine ? key(lo + j) : 0u, bin = (k >> shift) & ((1u << bits) - 1u);
            const bool in = j < mine && (k & high) == prefix;
            const uint32_t active = __ballot_sync(0xffffffffu, in);
            if (active == 0u) continue;
            const uint32_t leader = __ffs(active) - 1u, its = __shfl_sync(0xffffffffu, bin, leader);
            if (__all_sync(0xffffffffu, !in || bin == its)) {
                if (lane == leader) atomicAdd(&sh.bins[bin], (uint32_t)__popc(active));
            } else if (in) {
                atomicAdd(&sh.bins[bin], 1u);
            }
        }
        __syncthreads();
        static_assert(SELECT_BINS == 4 * SELECT_THREADS && SELECT_GROUPS == 64, "eight threads have a group, four bins each");
        {
            const uint4 x = *reinterpret_cast<const uint4*>(sh.bins + 4u * tid);
            uint32_t sum = x.x + x.y + x.z + x.w;
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            const uint32_t at = tc::smem_u32(&sh.groups_of[me][tid / 8u]);
            for (uint32_t c = tid & 7u; c < peers; c += 8u) tc::st_cluster(tc::map_to_rank(at, c), sum);
        }
        cluster_meet();
        if (warp == 0) {  // the group, from the top, two a lane
            uint32_t g0 = 0, g1 = 0;  // the lane's lower and upper group
            for (uint32_t c = 0; c < peers; ++c) {
                const uint2 x = *reinterpret_cast<const uint2*>(&sh.groups_of[c][SELECT_GROUPS - 2u * (lane + 1u)]);
                g0 += x.x, g1 += x.y;
            }
            uint32_t above = lanes_before(g0 + g1);
            if (above < want && above + g0 + g1 >= want) {
                const bool lower = above + g1 < want;
                sh.pick[0] = SELECT_GROUPS - 1u - 2u * lane - (lower ? 1u : 0u);
                sh.pick[1] = above + (lower ? g1 : 0u);
            }
        }
        __syncthreads();
        const uint32_t group = sh.pick[0];
        if (tid / 32u < peers) tc::st_cluster(tc::map_to_rank(tc::smem_u32(&sh.bins_of[me][lane]), tid / 32u), sh.bins[group * 32u + lane]);
        cluster_meet();
        if (warp == 0) {  // the bin in it, from the top
            uint32_t own = 0;
            for (uint32_t c = 0; c < peers; ++c) own += sh.bins_of[c][31u - lane];
            const uint32_t above = sh.pick[1] + lanes_before(own);
            if (above < want && above + own >= want) sh.pick[2] = 31u - lane, sh.pick[3] = want - above;
        }
        __syncthreads();
        const uint32_t in_group = sh.pick[2];
        prefix |= (group * 32u + in_group) << shift;
        want = sh.pick[3];
        const uint32_t members = lane < peers ? sh.bins_of[lane][in_group] : 0u, all_members = __reduce_add_sync(0xffffffffu, members);
        if (pass == 0 && all_members <= SELECT_LIST) {
            const uint32_t at = __reduce_add_sync(0xffffffffu, lane < me ? members : 0u);  // where this CTA's keys go in every CTA's list
            for (uint32_t j0 = 0; j0 < mine; j0 += SELECT_THREADS) {
                const uint32_t j = j0 + tid, k = j < mine ? key(lo + j) : 0u;
                if (j < mine && (k >> shift) == (prefix >> shift)) {
                    const uint32_t to = tc::smem_u32(sh.list + at + atomicAdd(&sh.found, 1u));
                    for (uint32_t c = 0; c < peers; ++c) tc::st_cluster(tc::map_to_rank(to, c), k);
                }
            }
            cluster_meet();
            // its lower 21 bits, 11 and 10 at a time
            static_assert(SELECT_BITS == 11, "21 bits are left");
#pragma unroll 1
            for (int low = 10; low >= 0; low -= 10) {
                const int width = low ? 11 : 10;
                *reinterpret_cast<uint4*>(sh.bins + 4u * tid) = make_uint4(0, 0, 0, 0);
                __syncthreads();
                for (uint32_t j = tid; j < all_members; j += SELECT_THREADS) {
                    const uint32_t k = sh.list[j];
                    if ((k >> (low + width)) == (prefix >> (low + width))) atomicAdd(&sh.bins[(k >> low) & ((1u << width) - 1u)], 1u);
                }
                __syncthreads();
                // thread t: four bins, from the top
                const uint32_t lowest = SELECT_BINS - 4u * (tid + 1u);
                const uint4 x = *reinterpret_cast<const uint4*>(sh.bins + lowest);
                const uint32_t own = x.x + x.y + x.z + x.w;
                uint32_t above = lanes_before(own);
                if (lane == 31u) sh.warps[warp].x = above + own;
                __syncthreads();
                above += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warps[lane].x : 0u);
                if (above < want && above + own >= want) {
                    uint32_t bin = lowest + 3u;
                    if (above + x.w < want) {
                        above += x.w, --bin;
                        if (above + x.z < want) {
                            above += x.z, --bin;
                            if (above + x.y < want) above += x.y, --bin;
                        }
                    }
                    sh.pick[2] = bin, sh.pick[3] = want - above;
                }
                __syncthreads();
                prefix |= sh.pick[2] << low;
                want = sh.pick[3];
            }
            break;
        }
    }

    uint4 count = make_uint4(0, 0, 0, 0);  // larger, equal below the new end; larger, equal behind it
    for (uint32_t e0 = wlo; e0 < whi; e0 += 32u) {
        const uint32_t e = e0 + lane, k = e < whi ? key(e) : 0u;
        const bool larger = e < whi && k > prefix, equal = e < whi && k == prefix, below = e < a.keep;
        count.x += __popc(__ballot_sync(0xffffffffu, larger && below)), count.y += __popc(__ballot_sync(0xffffffffu, equal && below));
        count.z += __popc(__ballot_sync(0xffffffffu, larger && !below)), count.w += __popc(__ballot_sync(0xffffffffu, equal && !below));
    }
    uint4 total;
    uint4 before = warps_before(count, sh.warps, &total);
    if (tid < peers) {
        const uint32_t to = tc::map_to_rank(tc::smem_u32(&sh.counts_of[me]), tid);
        tc::st_cluster(to, total.x), tc::st_cluster(to + 4u, total.y), tc::st_cluster(to + 8u, total.z), tc::st_cluster(to + 12u, total.w);
    }
    cluster_meet();  // the last word between the CTAs: any may leave after it
    {
        const uint4 other = lane < me ? sh.counts_of[lane] : make_uint4(0, 0, 0, 0);
        before.x += __reduce_add_sync(0xffffffffu, other.x), before.y += __reduce_add_sync(0xffffffffu, other.y);
        before.z += __reduce_add_sync(0xffffffffu, other.z), before.w += __reduce_add_sync(0xffffffffu, other.w);
    }
    // Entries below the end come before those behind it, so the ties, kept entries and holes before the warp follow from the four counts. As the first
    // `want` ties stay: below the end, kept = larger + min(ties, want).
    uint32_t ties = before.y + before.w, holes, late;
    {
        const uint32_t entries_below = min(wlo, a.keep);
        holes = entries_below - (before.x + min(before.y, want));
        const uint32_t ties_behind = before.w;  // only where the warp's entries begin behind the end are these counted, and then all ties below are before them
        late = before.z + (min(before.y + ties_behind, want) - min(before.y, want));
    }
    uint32_t* late_list = a.late + ((size_t)i * a.c.kv_heads + h) * a.keep;
    const uint32_t under = (1u << lane) - 1u;
    for (uint32_t e0 = wlo; e0 < whi; e0 += 32u) {
        const uint32_t e = e0 + lane, k = e < whi ? key(e) : 0u;
        const bool equal = e < whi && k == prefix, below = e < a.keep;
        const uint32_t tie_mask = __ballot_sync(0xffffffffu, equal);
        const bool stays = e < whi && (k > prefix || (equal && ties + __popc(tie_mask & under) < want));
        ties += __popc(tie_mask);
        const bool hole = e < whi && below && !stays, behind = stays && !below;
        const uint32_t hole_mask = __ballot_sync(0xffffffffu, hole), late_mask = __ballot_sync(0xffffffffu, behind);
        if (e < whi && below) plan[e] = stays ? e : EVICT_HOLE + holes + __popc(hole_mask & under);
        if (behind) late_list[late + __popc(late_mask & under)] = e;
        holes += __popc(hole_mask);
        late += __popc(late_mask);
    }
}

// Warp = MOVE_PLACES kept places of one kv head, looked up together, a lane each; four rows on their way at a time. In place a source lies behind the new end and a target before it, so
// that no copy reads what another writes. Bound by HBM and the chain plan, late list, page tables, rows.
constexpr uint32_t MOVE_PLACES = 8, MOVE_AT_ONCE = 4;
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a, uint32_t row_bytes, uint32_t elem, uint32_t vec) {
    pdl_wait();
    pdl_trigger();
    const uint32_t i = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31u, place0 = (blockIdx.x * 8u + (threadIdx.x >> 5)) * MOVE_PLACES;
    if (place0 >= a.keep) return;
    const uint32_t slot = a.seq[i];
    if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.new_len[i] = a.kept[i];
    const size_t list = ((size_t)i * a.c.kv_heads + h) * a.keep, base = ((size_t)slot * a.c.kv_heads + h) * a.ld;
    // lanes 0 .. MOVE_PLACES - 1 look a place up each
    uint32_t src = PAGED_NONE, from = PAGED_NONE, into = PAGED_NONE;
    const uint32_t place = place0 + lane;
    if (lane < MOVE_PLACES && place < a.keep) {
        src = a.plan[list + place];
        if (src != PAGED_NONE && src >= EVICT_HOLE) src = a.late[list + (src - EVICT_HOLE)];
        if (a.origin) a.origin[list + place] = src;
        if (src != PAGED_NONE) {
            const bool stays_put = a.in_place && src == place;
            if (!stays_put) {
                from = paged_page(a.c, slot, src), into = paged_page(a.to, slot, place);
                if (from == PAGED_NONE || into == PAGED_NONE) {
                    atomicOr(a.status, from == PAGED_NONE ? 1u : 2u);
                    from = PAGED_NONE;
                }
            }
            if (a.weights_out && (src != place || a.weights_out != a.weights)) a.weights_out[base + place] = a.weights[base + src];
            if (a.entry_pos_out && (src != place || a.entry_pos_out != a.entry_pos)) a.entry_pos_out[base + place] = a.entry_pos ? a.entry_pos[base + src] : src;
        }
    }
    // every lane with a place has its rows' offsets; MOVE_AT_ONCE of them move together
    const bool moving = from != PAGED_NONE;
    const size_t own_s = moving ? paged_row(a.c, from, h, src) * elem : 0, own_d = moving ? paged_row(a.to, into, h, place) * elem : 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, moving);
    for (uint32_t k0 = 0; k0 < MOVE_PLACES; k0 += MOVE_AT_ONCE) {
        if (((mask >> k0) & ((1u << MOVE_AT_ONCE) - 1u)) == 0u) continue;
        size_t s[MOVE_AT_ONCE], d[MOVE_AT_ONCE];
        bool moves[MOVE_AT_ONCE];
#pragma unroll
        for (uint32_t k = 0; k < MOVE_AT_ONCE; ++k) {
            moves[k] = (mask >> (k0 + k)) & 1u;
            s[k] = __shfl_sync(0xffffffffu, own_s, k0 + k), d[k] = __shfl_sync(0xffffffffu, own_d, k0 + k);
        }
        if (vec) {
            // 16-byte pieces of a key row, then of its value row
            const uint32_t half = row_bytes / 16u;
            for (uint32_t p = lane; p < 2u * half; p += 32u) {
                const bool value = p >= half;
                const uint32_t b = (value ? p - half : p) * 16u;
                const unsigned char* in = value ? a.c.v : a.c.k;
                unsigned char* out = value ? a.to.v : a.to.k;
                uint4 x[MOVE_AT_ONCE];
#pragma unroll
                for (uint32_t k = 0; k < MOVE_AT_ONCE; ++k)
                    if (moves[k]) x[k] = *reinterpret_cast<const uint4*>(in + s[k] + b);
#pragma unroll
                for (uint32_t k = 0; k < MOVE_AT_ONCE; ++k)
                    if (moves[k]) *reinterpret_cast<uint4*>(out + d[k] + b) = x[k];
            }
        } else {
#pragma unroll
            for (uint32_t k = 0; k < MOVE_AT_ONCE; ++k)
                for (uint32_t b = lane * 2u; moves[k] && b < row_bytes; b += 64u) {
                    *reinterpret_cast<uint16_t*>(a.to.k + d[k] + b) = *reinterpret_cast<const uint16_t*>(a.c.k + s[k] + b);
                    *reinterpret_cast<uint16_t*>(a.to.v + d[k] + b) = *reinterpret_cast<const uint16_t*>(a.c.v + s[k] + b);
                }
        }
    }
}

cudaError_t launch_select(const EvictArgs& a, uint32_t count, uint32_t peers, size_t smem, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(SELECT_CACHED * 8u));  // the same from every thread
    if (e == cudaSuccess && peers > 8u) e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.c.kv_heads * peers, count);
    cfg.blockDim = dim3(SELECT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = peers;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = m40_pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, evict_select_kernel, a);
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
    if (c->q_heads && c->q_out == c->q && c->ld && c->ld != wide) return -2;
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
    const size_t smem = (size_t)c->pairs * sizeof(float2);
    const uint32_t want = (uint32_t)(4 * ctx->sm_count) / c->rows;
    // a head's units of eight values lie on 16 bytes in every array, and turn as a whole or not
    const uintptr_t address = (uintptr_t)c->k | (uintptr_t)c->v | (c->q_heads ? (uintptr_t)c->q | (uintptr_t)c->q_out : 0);
    const bool eights = cache->head_dim % 8u == 0 && c->pairs % 4u == 0 && (address & 15u) == 0 && a.ld_q % 4u == 0 && a.ld_k % 4u == 0 && m40_paged_vec16(cache);
    const uint32_t threads = eights ? APPEND_THREADS : 256u, most = (uint32_t)((eights ? units / 4u : units) + threads - 1u) / threads;
    const dim3 grid(c->rows, want < 1u ? 1u : (want < most ? want : most));
    const bool f32 = cache->elem_dtype == M40LLM_DT_F32;
    void (*kernel)(AppendArgs) = eights ? (f32 ? paged_append_vec_kernel<float> : paged_append_vec_kernel<__half>)
                                        : (f32 ? paged_append_kernel<float> : paged_append_kernel<__half>);
    const cudaError_t e = m40_launch_dependent(kernel, grid, dim3(threads), smem, ctx->decode_stream, a);
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
    if (to->k == cache->k && to->table == cache->table && (to->v != cache->v || to->page_tokens != cache->page_tokens || to->max_pages != cache->max_pages)) return -2;
    if (to->elem_dtype != cache->elem_dtype) return -4;
    const size_t places = (size_t)c->count * cache->kv_heads * c->keep;  // below 2^62
    if (c->count > 65535u || places > PAGED_SCRATCH_MOST / 16u) return M40LLM_ERR_LIMIT;
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
    uint32_t* work = (uint32_t*)m40_ensure_scratch(ctx, 1, (2 * places + c->count) * sizeof(uint32_t), 0);
    if (!work) return -5;
    a.plan = work;
    a.late = work + places;
    a.kept = work + 2 * places;
    a.origin = c->origin;
    // as many CTAs for a list as fill the device once, with 512 entries or more each
    const uint64_t lists = (uint64_t)c->count * cache->kv_heads;
    uint32_t peers = 1u;
    while (peers < SELECT_CLUSTER && lists * peers * 2u <= (uint64_t)ctx->sm_count && a.bound > SELECT_THREADS * peers) peers *= 2u;
    // By the bound, not the lengths: lists far below it make their keys again in every pass (16 slots of 8 lists of 1025 to 1100 entries under a bound of 32768
    // 35.5 us, of 16384 31.4).
    const uint32_t per = (a.bound + peers - 1u) / peers;
    a.cached = per <= SELECT_CACHED ? per : 0u;
    cudaError_t e = launch_select(a, c->count, peers, (size_t)a.cached * 8u, ctx->decode_stream);
    if (e != cudaSuccess && peers > 8u) {  // a device that has no room for clusters of more than 8
        cudaGetLastError();
        peers = 8u;
        a.cached = (a.bound + peers - 1u) / peers <= SELECT_CACHED ? (a.bound + peers - 1u) / peers : 0u;
        e = launch_select(a, c->count, peers, (size_t)a.cached * 8u, ctx->decode_stream);
    }
    M40_COUNT_LAUNCH(ctx);
    if (e != cudaSuccess) return cudaGetLastError(), -3;
    const uint32_t elem = cache->elem_dtype == M40LLM_DT_F32 ? 4u : 2u;
    e = m40_launch_dependent(evict_move_kernel, dim3((c->keep + 8u * MOVE_PLACES - 1u) / (8u * MOVE_PLACES), cache->kv_heads, c->count), dim3(256), 0,
                             ctx->decode_stream, a, cache->head_dim * elem, elem, m40_paged_vec16(cache) && m40_paged_vec16(to) ? 1u : 0u);
    M40_COUNT_LAUNCH(ctx);
    if (e != cudaSuccess) return cudaGetLastError(), -3;
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // extern "C"
