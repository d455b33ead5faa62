// Log probabilities of given tokens with rank, entropy and the most likely alternatives: m40llm_logprobs_f32_async.
#include "common.cuh"
#include "tc_ptx.cuh"

namespace {

constexpr uint32_t LP_TOP_MAX = 64, LP_NONE = 0xffffffffu;
constexpr float LP_LOG2E = 1.4426950408889634f;

struct LogprobArgs {
    const float* logits;
    const uint32_t* tokens;
    float* logprob;
    uint32_t* rank;
    float* entropy;
    float* lse;
    uint32_t* top_ids;
    float* top_logprobs;
    uint32_t* status;
    uint32_t n, ld, top;
};

struct __align__(8) Candidate {
    float v;
    uint32_t i;
};
// the order of the list: larger values first, equal ones by index
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }  // NaN counts as -inf
// x relative to the row's largest value: where that is +inf, the values of +inf share the probability
__device__ __forceinline__ float against(float x, float top) { return x == top ? 0.0f : x - top; }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The row's results but for the list; ahead = values before the token's.
__device__ __forceinline__ void lp_store(const LogprobArgs& a, size_t row, float top, float s, float t, uint32_t token, float mine, uint32_t ahead) {
    const bool any = top > -INFINITY;
    const float rest = logf(s);
    if (a.lse) a.lse[row] = any ? top + rest : -INFINITY;
    if (a.entropy) a.entropy[row] = any ? rest - t / s : 0.0f;
    if (token < a.n) {
        if (a.logprob) a.logprob[row] = any ? against(mine, top) - rest : -INFINITY;
        if (a.rank) a.rank[row] = ahead + 1u;
    } else if (a.tokens) {
        if (a.logprob) a.logprob[row] = -INFINITY;
        if (a.rank) a.rank[row] = 0u;
        atomicOr(a.status, 8u);
    }
}
__device__ __forceinline__ void lp_list(const LogprobArgs& a, size_t row, uint32_t k, const Candidate& c, float top, float rest) {
    if (a.top_ids) a.top_ids[row * a.top + k] = c.i;
    if (a.top_logprobs) a.top_logprobs[row * a.top + k] = c.i == LP_NONE ? -INFINITY : against(c.v, top) - rest;
}

template <typename T, typename F>
__device__ __forceinline__ T warp_all(T v, F join) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ Candidate warp_best(Candidate c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Candidate u = {__shfl_xor_sync(0xffffffffu, c.v, o), __shfl_xor_sync(0xffffffffu, c.i, o)};
        if (before(u, c)) c = u;
    }
    return c;
}

constexpr uint32_t LP_LIST = 512;  // candidates that a CTA sorts by counting

// Larger is better, as f32; for maxima by integer reductions.
__device__ __forceinline__ uint32_t lp_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

// A sum of e = exp(x - m) and of e (x - m), m near the largest of its values (or -inf without any).
struct Sums {
    float m, s, t;
};
// `v` brought to reference m, the largest of the references that meet (a sum without values has the reference -inf).
__device__ __forceinline__ Sums moved(const Sums& v, float m) {
    const float d = against(v.m, m), e = exp2_fast(d * LP_LOG2E);
    return Sums{m, v.s * e, e > 0.0f ? (v.t + d * v.s) * e : 0.0f};
}
__device__ __forceinline__ Sums warp_joined(Sums v) {
    v = moved(v, lp_value(__reduce_max_sync(0xffffffffu, lp_key(v.m))));
    v.s = warp_sum(v.s);
    v.t = warp_sum(v.t);
    return v;
}
// two values at a time
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// What a CTA tells the first one of its cluster.
struct Share {
    Sums sums;
    uint32_t ahead;
    Candidate list[LP_TOP_MAX];
};
template <int WARPS>
struct LpShared {
    Candidate list[LP_LIST];
    Sums sums[WARPS];
    uint32_t ahead[WARPS], reach[WARPS], count, holders;
    uint16_t holder[32 * WARPS];
};

// A CTA's work on `count` values of a row, from value `first` on.
//   sums      every thread keeps a reference m, moved only when a value is more than 16 above it, so that exp(x - m) needs no second pass and no rescaling as a
//             rule; threads, warps and CTAs are joined by (s, t) -> (s e^(m - M), (t + (m - M) s) e^(m - M)). Entropy = log s - t / s.
//   rank      a value counts where it reaches the token's own, behind the token where it is larger.
//   list      of k: the k-th largest of the warps' maxima (more than the warps: the least of their r-th largest thread maxima, r = ceil(k / warps)) is
//             reached by at least k values, so the k largest are among those that reach it. These are few as a rule; what the threads hold whose maxima
//             reach it is looked at again (in L1 or L2), and they are sorted by counting who comes before whom. Where they are many (equal values, one thread's values above
//             all others, a mask that leaves 513 or more neighbours to fewer than k warps, whose bound is -inf), k rounds of a maximum over the block take their
//             place: a row of 32000 with 600 to 2000 neighbours left and k = 20 58 us instead of 8, 32 rows of 131077 67 instead of 11.
template <int T>
struct LpRow {
    static constexpr uint32_t WARPS = T / 32, AT_ONCE = 4;
    static constexpr float SLACK = 16.0f;
    const LogprobArgs& a;
    size_t row;
    const float* x;
    const float4* x4;
    uint32_t tid, first, count, token, split, head, fours, tail;
    float mine, reach, beyond;
    bool wanted, ranked;
    float m = -INFINITY, top = -INFINITY;
    uint64_t s2 = 0, t2 = 0;  // two sums each
    uint32_t above = 0;

    __device__ __forceinline__ LpRow(const LogprobArgs& args, size_t r, uint32_t from, uint32_t n, uint32_t tok, float tok_value)
        : a(args), row(r), tid(threadIdx.x), first(from), count(n), token(tok), mine(tok_value) {
        x = a.logits + row * a.ld + first;
        wanted = a.rank && token < a.n, ranked = wanted && mine < INFINITY;
        split = token < first ? 0u : token - first;  // the token's place among these values
        // behind a token of -inf come the values above it; before it all, NaN among them, which no comparison counts
        reach = mine > -INFINITY ? mine : NAN, beyond = ranked ? lp_value(lp_key(mine) + 1u) : INFINITY;
        if (ranked && mine == -INFINITY && tid == 0) above = min(split, count);
        // values [0, head) and [head + 4 * fours, count) one by one, the others by fours
        head = min((4u - (uint32_t)(((uintptr_t)x >> 2) & 3u)) & 3u, count), fours = (count - head) / 4u, tail = head + 4u * fours;
        x4 = reinterpret_cast<const float4*>(x + head);
    }
    __device__ __forceinline__ void move_to(float largest) {
        if (largest > m + SLACK) {
            const float d = m - largest, e = exp2_fast(d * LP_LOG2E);
            const float2 s = of_pair(s2), t = of_pair(t2);
            t2 = e > 0.0f ? pair_of((t.x + d * s.x) * e, (t.y + d * s.y) * e) : 0u;
            s2 = pair_of(s.x * e, s.y * e);
            m = largest;
        }
    }
    __device__ __forceinline__ void take2(float u, float v, uint64_t minus_m) {
        const float2 d = of_pair(add2(pair_of(u, v), minus_m));
        const uint64_t dd = pair_of(fmaxf(d.x, -200.0f), fmaxf(d.y, -200.0f));  // -inf and NaN: 0
        const float2 y = of_pair(mul2(dd, pair_of(LP_LOG2E, LP_LOG2E)));
        const uint64_t e = pair_of(exp2_fast(y.x), exp2_fast(y.y));
        s2 = add2(s2, e);
        t2 = fma2(e, dd, t2);
    }
    __device__ __forceinline__ void take_edges() {
        if (tid < head + (count - tail)) {  // at most six
            const uint32_t i = tid < head ? tid : tail + tid - head;
            const float v = clean(x[i]);
            top = fmaxf(top, v);
            move_to(v);
            take2(v, -INFINITY, pair_of(-m, -m));
            if (ranked) above += v >= (i < split ? reach : beyond);
        }
    }
    // the fours j0, j0 + T, ..
    __device__ __forceinline__ void take(const float4 (&v)[AT_ONCE], uint32_t j0) {
        float largest = -INFINITY;  // NaN falls out
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; ++k) largest = fmaxf(fmaxf(largest, fmaxf(v[k].x, v[k].y)), fmaxf(v[k].z, v[k].w));
        top = fmaxf(top, largest);
        move_to(largest);
        const uint64_t minus_m = pair_of(-m, -m);
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; ++k) take2(v[k].x, v[k].y, minus_m), take2(v[k].z, v[k].w, minus_m);
        if (ranked) {
            const uint32_t from = head + 4u * j0, to = from + 4u * (AT_ONCE - 1u) * T + 3u;
            if (to < split || from >= split) {  // all of them on one side of the token
                const float level = from >= split ? beyond : reach;
#pragma unroll
                for (uint32_t k = 0; k < AT_ONCE; ++k) above += v[k].x >= level, above += v[k].y >= level, above += v[k].z >= level, above += v[k].w >= level;
            } else {
#pragma unroll
                for (uint32_t k = 0; k < AT_ONCE; ++k) {
                    const uint32_t i = from + 4u * k * T;
                    above += v[k].x >= (i < split ? reach : beyond), above += v[k].y >= (i + 1u < split ? reach : beyond);
                    above += v[k].z >= (i + 2u < split ? reach : beyond), above += v[k].w >= (i + 3u < split ? reach : beyond);
                }
            }
        }
    }
    // The CTAs' lists meet in the first one of a cluster, where a candidate's place is its place in its own list plus what binary search finds in the others.
    __device__ __forceinline__ void finish(LpShared<WARPS>& sh, uint32_t me, uint32_t peers, Share* share) {
        const uint32_t lane = tid & 31u, warp = tid >> 5;
        Sums sums;
        const uint32_t full = max(1u, min(WARPS, fours / 32u));  // warps whose threads all have values, or the first
        {
            const float2 s = of_pair(s2), t = of_pair(t2);
            sums = warp_joined(moved(Sums{m, s.x + s.y, t.x + t.y}, top));  // its reference is the warp's largest value from here on
            uint32_t key = lp_key(top), best = __reduce_max_sync(0xffffffffu, key);
            // more alternatives than warps: the r-th largest of the warp's maxima (equal ones one by one)
            const uint32_t r = (a.top + full - 1u) / full;
            for (uint32_t i = 1; i < r; ++i) {
                const uint32_t holder = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1u;
                if (lane == holder) key = 0u;
                best = __reduce_max_sync(0xffffffffu, key);
            }
            above = __reduce_add_sync(0xffffffffu, above);
            if (lane == 0) sh.sums[warp] = sums, sh.ahead[warp] = above, sh.reach[warp] = best;
        }
        __syncthreads();
        sums = warp_joined(lane < WARPS ? sh.sums[lane] : Sums{-INFINITY, 0.0f, 0.0f});
        above = __reduce_add_sync(0xffffffffu, lane < WARPS ? sh.ahead[lane] : 0u);
        float bound = sums.m;
        if (a.top > 1u) {
            const uint32_t key = lane < WARPS ? sh.reach[lane] : 0u;
            uint32_t least = lp_key(-INFINITY);
            if (a.top <= full) {  // the k-th largest of the warps' maxima, by the upper half of its bits
                uint32_t prefix = 0u;
                for (uint32_t bit = 0x80000000u; bit > 0x8000u; bit /= 2u)
                    if ((uint32_t)__popc(__ballot_sync(0xffffffffu, lane < full && key >= (prefix | bit))) >= a.top) prefix |= bit;
                least = max(least, prefix);
            } else {
                least = max(least, __reduce_min_sync(0xffffffffu, lane < full ? key : 0xffffffffu));
            }
            bound = lp_value(least);
        }
        if (a.top) {
            const auto meet = [&](uint32_t i, float u) {
                if (u >= bound && u > -INFINITY) {
                    const uint32_t at = atomicAdd(&sh.count, 1u);
                    if (at < LP_LIST) sh.list[at] = Candidate{u, first + i};
                }
            };
            const auto meet_four = [&](uint32_t j) {
                const float4 v = x4[j];
                const uint32_t i = head + 4u * j;
                if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bound) meet(i, v.x), meet(i + 1u, v.y), meet(i + 2u, v.z), meet(i + 3u, v.w);
            };
            const uint32_t each = (fours + T - 1u) / T;
            const bool holds = top >= bound && top > -INFINITY;
            if (holds && tid < head + (count - tail)) {
                const uint32_t i = tid < head ? tid : tail + tid - head;
                meet(i, x[i]);
            }
            if (each <= 12u) {
                if (holds)
#pragma unroll 4
                    for (uint32_t j = tid; j < fours; j += T) meet_four(j);
            } else {
                // many fours a thread: all threads look at the holders' (each at its own, one held up the others for up to 5600 cycles: 64.6 against 54 us for 2048
                // rows of 32000; with few, the barrier costs more: 32 rows of 131077 18 against 22 us)
                if (holds) sh.holder[atomicAdd(&sh.holders, 1u)] = (uint16_t)tid;
                __syncthreads();
                const uint32_t holders = sh.holders;
                for (uint32_t w = tid; w < holders * each; w += T) {
                    const uint32_t q = w / each, j = sh.holder[q] + (w - q * each) * T;
                    if (j < fours) meet_four(j);
                }
            }
        }
        // what the sums do not tell: infinities share the probability; the rank of an infinite value is counted value by value
        const bool infinite = sums.m == INFINITY, recount = wanted && !ranked;
        if (infinite || recount) {
            uint32_t n_inf = 0, n_ahead = 0;
            for (uint32_t i = tid; i < count; i += T) {
                const float v = clean(x[i]);
                n_inf += v == INFINITY;
                n_ahead += v > mine || (v == mine && first + i < token);
            }
            n_inf = __reduce_add_sync(0xffffffffu, n_inf);
            n_ahead = __reduce_add_sync(0xffffffffu, n_ahead);
            __syncthreads();  // the sums and counts above have been read
            if (lane == 0) sh.reach[warp] = n_inf, sh.ahead[warp] = n_ahead;
            __syncthreads();
            if (infinite) sums.s = (float)__reduce_add_sync(0xffffffffu, lane < WARPS ? sh.reach[lane] : 0u), sums.t = 0.0f;
            if (recount) above = __reduce_add_sync(0xffffffffu, lane < WARPS ? sh.ahead[lane] : 0u);
        }
        __syncthreads();
        const uint32_t found = sh.count;
        const bool alone = peers == 1u;
        const float rest = logf(sums.s);
        uint32_t remote = 0;  // this CTA's share, in the first one's memory
        if (alone) {
            if (tid == 0) lp_store(a, row, sums.m, sums.s, sums.t, token, mine, above);
        } else {
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            remote = tc::map_to_rank(tc::smem_u32(share + me), 0);
            if (tid == 0) {
                tc::st_cluster(remote + offsetof(Share, sums.m), __float_as_uint(sums.m));
                tc::st_cluster(remote + offsetof(Share, sums.s), __float_as_uint(sums.s));
                tc::st_cluster(remote + offsetof(Share, sums.t), __float_as_uint(sums.t));
                tc::st_cluster(remote + offsetof(Share, ahead), above);
            }
        }
        const auto put = [&](uint32_t k, const Candidate& c) {
            if (alone) {
                lp_list(a, row, k, c, sums.m, rest);
            } else {
                tc::st_cluster(remote + offsetof(Share, list) + k * 8u, __float_as_uint(c.v));
                tc::st_cluster(remote + offsetof(Share, list) + k * 8u + 4u, c.i);
            }
        };
        if (found <= LP_LIST) {
            // four threads count for one candidate
            for (uint32_t c = tid / 4u; c < ((found + 7u) & ~7u); c += T / 4u) {
                const Candidate own = sh.list[min(c, LP_LIST - 1u)];
                uint32_t place = 0;
                for (uint32_t j = tid & 3u; j < found; j += 4u) place += before(sh.list[j], own);
                place += __shfl_xor_sync(0xffffffffu, place, 1);
                place += __shfl_xor_sync(0xffffffffu, place, 2);
                if ((tid & 3u) == 0 && c < found && place < a.top) put(place, own);
            }
            for (uint32_t k = found + tid; k < a.top; k += T) put(k, Candidate{-INFINITY, LP_NONE});
        } else {
            Candidate prev = {INFINITY, 0u};
            for (uint32_t r = 0; r < a.top; ++r) {
                Candidate best = {-INFINITY, LP_NONE};
                for (uint32_t i = tid; i < count; i += T) {
                    const Candidate c = {clean(x[i]), first + i};
                    if (c.v > -INFINITY && (r == 0 || before(prev, c)) && before(c, best)) best = c;
                }
                best = warp_best(best);
                __syncthreads();
                if (lane == 0) sh.list[warp] = best;
                __syncthreads();
                best = warp_best(lane < WARPS ? sh.list[lane] : Candidate{-INFINITY, LP_NONE});
                if (tid == 0) put(r, best);
                prev = best;
            }
        }
        if (alone) return;
        tc::cluster_sync_all();
        if (me != 0) return;

        sums = warp_joined(lane < peers ? share[lane].sums : Sums{-INFINITY, 0.0f, 0.0f});
        above = __reduce_add_sync(0xffffffffu, lane < peers ? share[lane].ahead : 0u);
        if (tid == 0) lp_store(a, row, sums.m, sums.s, sums.t, token, mine, above);
        const float rest_all = logf(sums.s);
        for (uint32_t q = tid; q < peers * a.top; q += T) {
            const uint32_t c = q / a.top, k = q - c * a.top;
            const Candidate own = share[c].list[k];
            uint32_t lo[8], place = k;  // the values of the other lists that come before this one; the lists' empty places end them
#pragma unroll
            for (uint32_t o = 0; o < 8u; ++o) lo[o] = 0;
            const bool empty = own.i == LP_NONE;
            for (uint32_t step = 64u; step; step /= 2u)
#pragma unroll
                for (uint32_t o = 0; o < 8u; ++o)
                    if (o < peers && lo[o] + step <= a.top) {
                        const Candidate u = share[o].list[lo[o] + step - 1u];
                        if (u.i != LP_NONE && (empty || before(u, own))) lo[o] += step;
                    }
#pragma unroll
            for (uint32_t o = 0; o < 8u; ++o)  // an empty place comes behind every value and behind the empty places of the lists before its own
                if (o < peers && o != c) place += empty && o < c ? a.top : lo[o];
            if (place < a.top) lp_list(a, row, place, own, sums.m, rest_all);
        }
    }
};

// Cluster = one row (one CTA as a rule), CTA c has the values [c * per, (c + 1) * per). The row is read once, with four 16-byte loads of a thread on their way
// together. Bound by a chain of memory and barrier latencies.
template <int T, int CTAS>
__global__ void __launch_bounds__(T, CTAS) logprobs_kernel(LogprobArgs a, uint32_t per) {
    __shared__ Share s_share[8];
    __shared__ LpShared<T / 32> sh;
    pdl_wait();
    pdl_trigger();
    uint32_t peers;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(peers));
    const uint32_t me = tc::cluster_rank(), tid = threadIdx.x, first = me * per;  // first < n
    const size_t row = blockIdx.x / peers;
    if (peers > 1u) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // every CTA of the cluster is there
    if (tid == 0) sh.count = 0u, sh.holders = 0u;
    const uint32_t token = a.tokens ? a.tokens[row] : LP_NONE;
    LpRow<T> r(a, row, first, min(per, a.n - first), token, token < a.n ? clean(a.logits[row * a.ld + token]) : INFINITY);
    r.take_edges();
    constexpr uint32_t AT_ONCE = LpRow<T>::AT_ONCE;
    uint32_t j0 = tid;
    for (; j0 + (AT_ONCE - 1u) * T < r.fours; j0 += AT_ONCE * T) {
        float4 v[AT_ONCE];
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; ++k) v[k] = r.x4[j0 + k * T];
        r.take(v, j0);
    }
    if (j0 < r.fours) {
        float4 v[AT_ONCE];
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; ++k) v[k] = j0 + k * T < r.fours ? r.x4[j0 + k * T] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        r.take(v, j0);
    }
    r.finish(sh, me, peers, s_share);
}

template <int T, int CTAS>
cudaError_t launch_logprobs(const LogprobArgs& a, uint32_t rows, uint32_t peers, uint32_t per, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * peers);
    cfg.blockDim = dim3(T);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = peers;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = m40_pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, CTAS>, a, per);
}

}  // namespace

extern "C" int m40llm_logprobs_f32_async(M40llmCudaContext* ctx, const M40llmLogprobs* c) {
    if (!ctx || !c || !c->logits || ((c->logprob || c->rank) && !c->tokens)) return -1;
    if (c->rows == 0 || c->n == 0 || (c->ld && c->ld < c->n)) return -2;
    if (c->top > LP_TOP_MAX || c->n > (1u << 30) || c->rows > (1u << 27)) return M40LLM_ERR_LIMIT;
    if (m40_ensure_device(ctx) != 0) return -1;
    const LogprobArgs a = {(const float*)c->logits, c->tokens, (float*)c->logprob, c->rank, (float*)c->entropy, (float*)c->lse, c->top_ids,
                           (float*)c->top_logprobs, ctx->d_status, c->n, c->ld ? c->ld : c->n,
                           c->top_ids || c->top_logprobs ? c->top : 0u};
    // More rows than SMs: a CTA of 256 threads each, five per SM (2048 rows of 32000 values 50.4 us, 52 on other B200s, 300 rows 14.2; with 512 threads 54.7 and 14.6, with 128
    // and twice the loads 48.6 and 19.6). Else 1024 threads (80 rows 7.3 us against 8.5), and up to 8 CTAs that have 32768 values or more (a row of 32000: one
    // CTA 7.4 to 7.9 us, two 8.9, four 9.5; of 64000: two 10.0, four 9.5, eight 11.0).
    const uint64_t sms = (uint64_t)ctx->sm_count;
    uint32_t peers = 1u;
    while (peers < 8u && peers * 2ull * c->rows <= sms && c->n > 32768u * peers) peers *= 2u;
    const uint32_t per = (((c->n + peers - 1u) / peers) + 3u) & ~3u;
    peers = (c->n + per - 1u) / per;  // no CTA without values
    const cudaError_t e = c->rows <= sms ? launch_logprobs<1024, 1>(a, c->rows, peers, per, ctx->decode_stream)
                                         : launch_logprobs<256, 5>(a, c->rows, peers, per, ctx->decode_stream);
    M40_COUNT_LAUNCH(ctx);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return -3;
    }
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
