// Log probabilities of given tokens, entropy and the best alternatives of rows of fp16 logits.
//
//   y = x / temperature, m = max y, S = sum exp(y - m)
//   logprob(i) = (y_i - m) - ln S,   entropy = ln S - sum (y - m) exp(y - m) / S
#include <cfloat>
#include <cmath>

#include "common.hpp"

#define LP_THREADS 256
#define LP_WAVES (LP_THREADS / 64)
#define LP_MAX_TOP LLM_LOGPROBS_MAX_TOP
#define LP_MAX_IDS LLM_LOGPROBS_MAX_IDS

struct LpArgs {
    const half_t *x;
    size_t ld;
    int vocab, n_ids, k;
    float inv_t;
    const int32_t *ids;
    float *logprob, *entropy, *top;
    int32_t *top_ids;
};

// One workgroup per row.
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const LpArgs a) {
    __shared__ float red[2][LP_WAVES];
    __shared__ unsigned long long best[LP_WAVES];
    const size_t row = blockIdx.x;
    const half_t *x = a.x + row * a.ld;
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    float m = -INFINITY;
    bool bad = false;
    for (int i = tid; i < a.vocab; i += LP_THREADS) {
        const float v = (float)x[i];
        bad |= !(v < INFINITY);
        m = fmaxf(m, v);
    }
    m = wave_max(m);
    if (__builtin_amdgcn_ballot_w64(bad)) m = NAN;
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = red[0][0];
    for (int w = 1; w < LP_WAVES; ++w) m = (m != m || red[0][w] != red[0][w]) ? NAN : fmaxf(m, red[0][w]);
    __syncthreads();
    const bool invalid = m != m, none = m == -INFINITY;
    const float m0 = none ? 0.f : m;
    float s = 0.f, t = 0.f;
    for (int i = tid; i < a.vocab; i += LP_THREADS) {
        const float y = ((float)x[i] - m0) * a.inv_t, e = __expf(y);
        s += e;
        t += fmaxf(y, -FLT_MAX) * e;
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) {
        red[0][wave] = s;
        red[1][wave] = t;
    }
    __syncthreads();
    s = t = 0.f;
    for (int w = 0; w < LP_WAVES; ++w) {
        s += red[0][w];
        t += red[1][w];
    }
    const float log_s = none ? 0.f : logf(s);
    if (tid == 0) a.entropy[row] = invalid ? NAN : none ? 0.f : log_s - t / s;
    if (tid < a.n_ids) {
        const int id = a.ids[row * a.n_ids + tid];
        float lp = NAN;
        if (id >= 0 && id < a.vocab && !invalid) lp = ((float)x[id] - m0) * a.inv_t - log_s;
        a.logprob[row * a.n_ids + tid] = lp;
    }
    unsigned long long below = ~0ull;
    for (int r = 0; r < a.k; ++r) {
        unsigned long long c = 0ull;
        for (int i = tid; i < a.vocab && !invalid; i += LP_THREADS) {
            const half_t h = x[i];
            if ((float)h == -INFINITY) continue;
            const unsigned long long p = pack_candidate(h, i);
            if (p < below && p > c) c = p;
        }
        for (int o = 32; o; o >>= 1) {
            const unsigned long long q = __shfl_xor(c, o);
            c = q > c ? q : c;
        }
        __syncthreads();
        if (lane == 0) best[wave] = c;
        __syncthreads();
        for (int w = 0; w < LP_WAVES; ++w) c = best[w] > c ? best[w] : c;
        below = c;
        if (tid == 0) {
            const int id = c ? (int)(0xffffffffu - (uint32_t)c) : -1;
            a.top_ids[row * a.k + r] = id;
            a.top[row * a.k + r] = invalid ? NAN : id < 0 ? -INFINITY : ((float)x[id] - m0) * a.inv_t - log_s;
        }
    }
}

extern "C" {

size_t llm_logprobs_workspace_bytes(int rows, int vocab, int k) {
    (void)rows, (void)vocab, (void)k;
    return 16;
}

int llm_logprobs(const uint16_t *logits, int ld, int rows, int vocab, float temperature, const int32_t *ids, int n_ids,
                 float *logprob, float *entropy, int k, int32_t *top_ids, float *top_logprob, void *workspace, llm_stream_t stream) {
    LLM_REQUIRE(rows >= 0 && vocab >= 1 && ld >= vocab, "llm_logprobs: %d rows of %d logits, ld=%d", rows, vocab, ld);
    LLM_REQUIRE(temperature > 0.f && temperature <= FLT_MAX && 1.f / temperature <= FLT_MAX, "llm_logprobs: temperature %g", (double)temperature);
    LLM_REQUIRE(n_ids >= 0 && n_ids <= LP_MAX_IDS, "llm_logprobs: %d given tokens per row (0..%d)", n_ids, LP_MAX_IDS);
    LLM_REQUIRE(k >= 0 && k <= LP_MAX_TOP && k <= vocab, "llm_logprobs: top %d of %d (at most %d)", k, vocab, LP_MAX_TOP);
    LLM_REQUIRE(logits && entropy && workspace && (n_ids == 0 || (ids && logprob)) && (k == 0 || (top_ids && top_logprob)),
                "llm_logprobs: null pointer");
    LLM_REQUIRE(((uintptr_t)logits & 1u) == 0 && aligned16(workspace) &&
                    (((uintptr_t)ids | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_logprob) & 3u) == 0,
                "llm_logprobs: logits must be aligned to 2 bytes, the workspace to 16, the others to 4");
    if (rows == 0) return LLM_OK;
    const LpArgs a = {(const half_t *)logits, (size_t)ld, vocab, n_ids, k, 1.f / temperature, ids, logprob, entropy, top_logprob, top_ids};
    logprobs_kernel<<<dim3(rows), dim3(LP_THREADS), 0, (hipStream_t)stream>>>(a);
    LLM_LAUNCH_CHECK("logprobs_kernel");
    return LLM_OK;
}

} // extern "C"
