// Log probabilities of given tokens with rank, entropy and the most likely alternatives: m40llm_logprobs_f32_async.
#include "common.cuh"

namespace {

constexpr uint32_t LP_THREADS = 1024, LP_TOP_MAX = 64, LP_NONE = 0xffffffffu;

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

struct Candidate {
    float v;
    uint32_t i;
};
// the order of the list: larger values first, equal ones by index
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ float clean(float x) { return isnan(x) ? -INFINITY : x; }
// x relative to the row's largest value: where that is +inf, the values of +inf share the probability
__device__ __forceinline__ float against(float x, float top) { return x == top ? 0.0f : x - top; }

template <typename T, typename F>
__device__ __forceinline__ T block_all(T v, T* red, F join) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        T u = v;
        u = __shfl_xor_sync(0xffffffffu, v, o);
        v = join(v, u);
    }
    __syncthreads();
    if ((threadIdx.x & 31u) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (uint32_t w = 1; w < LP_THREADS / 32; ++w) v = join(v, red[w]);
    return v;
}

// CTA = one row: largest value; sums of e = exp(x - top) and e (x - top); then one pass per alternative.
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(LogprobArgs a) {
    __shared__ float redf[32];
    __shared__ uint32_t redu[32];
    __shared__ Candidate redc[32];
    pdl_wait();
    pdl_trigger();
    const size_t row = blockIdx.x;
    const uint32_t tid = threadIdx.x;
    const float* x = a.logits + row * a.ld;
    const auto add = [](float p, float q) { return p + q; };
    float top = -INFINITY;
    for (uint32_t i = tid; i < a.n; i += LP_THREADS) top = fmaxf(top, clean(x[i]));
    top = block_all(top, redf, [](float p, float q) { return fmaxf(p, q); });
    const uint32_t token = a.tokens ? a.tokens[row] : LP_NONE;
    const float mine = token < a.n ? clean(x[token]) : -INFINITY;
    float s = 0.0f, t = 0.0f;
    uint32_t ahead = 0;
    for (uint32_t i = tid; i < a.n; i += LP_THREADS) {
        const float v = clean(x[i]), d = against(v, top), e = expf(d);
        s += e;
        if (e > 0.0f) t += e * d;
        ahead += v > mine || (v == mine && i < token);
    }
    s = block_all(s, redf, add);
    t = block_all(t, redf, add);
    ahead = block_all(ahead, redu, [](uint32_t p, uint32_t q) { return p + q; });
    const bool any = top > -INFINITY;
    const float rest = logf(s);
    if (tid == 0) {
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
    Candidate last = {INFINITY, 0u};
    bool started = false;
    for (uint32_t k = 0; k < a.top; ++k) {
        Candidate best = {-INFINITY, LP_NONE};
        for (uint32_t i = tid; i < a.n; i += LP_THREADS) {
            const Candidate c = {clean(x[i]), i};
            if ((!started || before(last, c)) && c.v > -INFINITY && before(c, best)) best = c;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Candidate u = {__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)};
            if (before(u, best)) best = u;
        }
        __syncthreads();
        if ((tid & 31u) == 0) redc[tid >> 5] = best;
        __syncthreads();
        best = redc[0];
        for (uint32_t w = 1; w < LP_THREADS / 32; ++w)
            if (before(redc[w], best)) best = redc[w];
        if (tid == 0) {
            if (a.top_ids) a.top_ids[row * a.top + k] = best.i;
            if (a.top_logprobs) a.top_logprobs[row * a.top + k] = best.i == LP_NONE ? -INFINITY : against(best.v, top) - rest;
        }
        last = best;
        started = true;
    }
}

}  // namespace

extern "C" int m40llm_logprobs_f32_async(M40llmCudaContext* ctx, const M40llmLogprobs* c) {
    if (!ctx || !c || !c->logits || ((c->logprob || c->rank) && !c->tokens)) return -1;
    if (c->rows == 0 || c->n == 0 || (c->ld && c->ld < c->n)) return -2;
    if (c->top > LP_TOP_MAX) return M40LLM_ERR_LIMIT;
    if (m40_ensure_device(ctx) != 0) return -1;
    const LogprobArgs a = {(const float*)c->logits, c->tokens, (float*)c->logprob, c->rank, (float*)c->entropy, (float*)c->lse, c->top_ids,
                           (float*)c->top_logprobs, ctx->d_status, c->n, c->ld ? c->ld : c->n,
                           c->top_ids || c->top_logprobs ? c->top : 0u};
    const cudaError_t e = m40_launch_dependent(logprobs_kernel, dim3(c->rows), dim3(LP_THREADS), 0, ctx->decode_stream, a);
    M40_COUNT_LAUNCH(ctx);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -3;
}
