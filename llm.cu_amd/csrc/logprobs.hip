// Log probabilities of given tokens, entropy and the best alternatives of rows of fp16 logits.
//
//   y = x / temperature, m = max y, S = sum exp(y - m)
//   logprob(i) = (y_i - m) - ln S,   entropy = ln S - sum (y - m) exp(y - m) / S
//
// One pass over the logits: a row is cut into chunks, one workgroup holds a chunk in registers, takes the sums relative to each
// wavefront's own maximum (no barrier between the loads and the exponentials) and picks the chunk's k best; the workgroup of a
// row that finishes last joins the chunks.  Exponentials are base 2: 2^((x - m) c) with c = log2(e) / temperature, x - m exact
// in fp32 for fp16 values of similar size, so nothing is lost at large logits or low temperatures.
//
// The k best (k <= 32) of a chunk without a sort: the k-th largest of the 64 lane maxima of a wavefront is a lower bound of the
// chunk's k-th largest logit, found by bisection on 16-bit order keys (ballot and bit count, 16 steps); the few logits from
// there up (about 1.2 k in random data) are listed in LDS and ranked by counting.  A listed logit is one 32-bit word, order key
// above the complement of its place, so that a larger word is a larger logit or an equal one further in front.
#include <cfloat>
#include <cmath>

#include "common.hpp"

#define LP_THREADS 256
#define LP_WAVES (LP_THREADS / 64)
#define LP_MAX_TOP LLM_LOGPROBS_MAX_TOP
#define LP_MAX_IDS LLM_LOGPROBS_MAX_IDS
#define LP_MAX_CHUNKS 64       // of a row: one lane each when they are joined
#define LP_MAX_LOADS 8         // 16-byte loads per thread and chunk: 16384 logits
#define LP_MAX_VOCAB (LP_MAX_CHUNKS * LP_THREADS * 8 * LP_MAX_LOADS)
#define LP_SLICE 4096          // rows per launch: a counter each at the front of the workspace
#define LP_MERGE (LP_MAX_CHUNKS * LP_MAX_TOP / LP_THREADS) // listed logits per thread when chunks are joined
#define LP_LOWEST 0x0400u      // order key of -65504, the lowest logit that has a probability

struct LpArgs {
    const half_t *x;
    size_t ld;
    int vocab, n_ids, k, chunks;
    float inv_t;
    const int32_t *ids;
    float *logprob, *entropy, *top;
    int32_t *top_ids;
    int *counters;
    uint32_t *stats;    // [row][chunk][4]: m, S, sum y 2^y (relative to m, base 2) as bits
    uint32_t *listed;   // [row][chunk][k]
};

struct LpStats {
    float m, s, t;
};

// eight logits from any element of a row
__device__ __forceinline__ half8_t lp_load8(const half_t *p) {
    half8_t v;
    __builtin_memcpy(&v, p, sizeof v);
    return v;
}

__device__ __forceinline__ uint32_t lp_key(half_t h) { return f16_order_key(__builtin_bit_cast(uint16_t, h)); }
__device__ __forceinline__ half_t lp_value(uint32_t key) { // the logit of an order key (+0 for either zero)
    return __builtin_bit_cast(half_t, (uint16_t)(key >= 0x8000u ? key - 0x8000u : 0xffffu - key));
}

__device__ __forceinline__ void lp_put(uint32_t *p, uint32_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint32_t lp_get(const uint32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// a part's sums relative to a larger maximum M
__device__ __forceinline__ LpStats lp_rebase(LpStats p, float M, float c) {
    if (p.s == 0.f) return {M, 0.f, 0.f}; // nothing in this part (its maximum is -inf)
    const float d = (p.m - M) * c, f = __builtin_amdgcn_exp2f(d);
    return {M, f * p.s, f == 0.f ? 0.f : f * (p.t + d * p.s)}; // d may be -inf at the lowest temperatures
}

// k-th largest of the lanes' keys (0: fewer than k lanes have one)
__device__ __forceinline__ uint32_t lp_kth_key(uint32_t key, int k) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 15; bit >= 0; --bit) {
        const uint32_t trial = t | 1u << bit;
        if (__popcll(__builtin_amdgcn_ballot_w64(key >= trial)) >= k) t = trial;
    }
    return t;
}

__device__ __forceinline__ uint32_t lp_wave_max(uint32_t v) {
    for (int o = 32; o; o >>= 1) {
        const uint32_t q = (uint32_t)__shfl_xor((int)v, o);
        v = q > v ? q : v;
    }
    return v;
}

// The k largest of the n distinct words in list, largest first, into best (zeros behind the last one).  All threads call it;
// best is ready behind the barrier it ends with.
__device__ __forceinline__ void lp_rank(const uint32_t *list, int n, int k, uint32_t *best, uint32_t *red) {
    const int tid = threadIdx.x;
    if (tid < k) best[tid] = 0u;
    __syncthreads();
    if (n <= 2 * LP_THREADS) {
        for (int i = tid; i < n; i += LP_THREADS) {
            const uint32_t v = list[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > v;
            if (rank < k) best[rank] = v;
        }
        __syncthreads();
        return;
    }
    uint32_t below = 0xffffffffu; // many words: their maximum, k times
    for (int r = 0; r < k; ++r) {
        uint32_t v = 0;
        for (int i = tid; i < n; i += LP_THREADS) {
            const uint32_t w = list[i];
            v = w < below && w > v ? w : v;
        }
        v = lp_wave_max(v);
        if (tid % 64 == 0) red[tid / 64] = v;
        __syncthreads();
        for (int w = 0; w < LP_WAVES; ++w) v = red[w] > v ? red[w] : v;
        if (tid == 0) best[r] = v;
        below = v;
        __syncthreads();
        if (v == 0) break;
    }
}

template <int NL>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const LpArgs a) {
    constexpr int CHUNK = LP_THREADS * 8 * NL;
    // A lane whose maximum is below the bound lists nothing, and fewer than k lanes of a wavefront have a maximum above it: more
    // than this many logits above the bound cannot be.
    constexpr int LIST = (LP_MAX_TOP * 8 * NL * LP_WAVES > LP_MAX_CHUNKS * LP_MAX_TOP) ? LP_MAX_TOP * 8 * NL * LP_WAVES : LP_MAX_CHUNKS * LP_MAX_TOP;
    __shared__ uint32_t list[LIST], best[LP_MAX_TOP], red[LP_WAVES], listed_n;
    __shared__ float part[LP_WAVES][3];
    __shared__ int is_last;
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, chunk = blockIdx.x, k = a.k;
    const size_t row = blockIdx.y;
    const half_t *x = a.x + row * a.ld;
    const float c = a.inv_t * 1.44269504088896341f;

    // ---- 1. the chunk into registers, -inf behind the end of the row --------------------------------------------------
    const half_t ninf = __builtin_bit_cast(half_t, (uint16_t)0xfc00u);
    half8_t v[NL];
#pragma unroll
    for (int u = 0; u < NL; ++u) {
        const int i = chunk * CHUNK + (u * LP_THREADS + tid) * 8;
        if (i + 8 <= a.vocab) {
            v[u] = lp_load8(x + i);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] = i + e < a.vocab ? x[i + e] : ninf;
        }
    }
    // ---- 2. the lane's and the wavefront's maximum, the sums relative to the latter -----------------------------------
    half8_t m8 = v[0];
#pragma unroll
    for (int u = 1; u < NL; ++u) m8 = __builtin_elementwise_max(m8, v[u]);
    half_t lane_max = ninf; // a NaN loses against any number here; the sums find it
#pragma unroll
    for (int e = 0; e < 8; ++e) lane_max = m8[e] > lane_max ? m8[e] : lane_max;
    LpStats st = {wave_max((float)lane_max), 0.f, 0.f};
    {
        const float m0 = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
        for (int u = 0; u < NL; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = ((float)v[u][e] - m0) * c, p = __builtin_amdgcn_exp2f(y);
                st.s += p;
                st.t = fmaf(fmaxf(y, -FLT_MAX), p, st.t); // -inf times zero is zero here; a NaN is in p already
            }
        st.s = wave_sum(st.s);
        st.t = wave_sum(st.t);
    }
    if (lane == 0) {
        part[wave][0] = st.m;
        part[wave][1] = st.s;
        part[wave][2] = st.t;
    }
    // ---- 3. the k best of the chunk ------------------------------------------------------------------------------------
    if (k > 0) {
        uint32_t bound = lane_max == ninf ? 0u : lp_key(lane_max);
        bound = k == 1 ? lp_wave_max(bound) : lp_kth_key(bound, k);
        if (lane == 0) red[wave] = bound;
        if (tid == 0) listed_n = 0u;
    }
    __syncthreads();
    float M = part[0][0];
#pragma unroll
    for (int w = 1; w < LP_WAVES; ++w) M = fmaxf(M, part[w][0]);
    st = {M, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w) {
        const LpStats p = lp_rebase({part[w][0], part[w][1], part[w][2]}, M, c);
        st.s += p.s;
        st.t += p.t;
    }
    if (k > 0) {
        uint32_t bound = LP_LOWEST; // no logit of probability zero
#pragma unroll
        for (int w = 0; w < LP_WAVES; ++w) bound = red[w] > bound ? red[w] : bound;
        const half_t bv = lp_value(bound);
        auto word = [&](int u, int e) { return lp_key(v[u][e]) << 16 | (uint32_t)(0xffff - ((u * LP_THREADS + tid) * 8 + e)); };
        if (lane_max >= bv) {
#pragma unroll
            for (int u = 0; u < NL; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (v[u][e] >= bv) {
                        const uint32_t at = atomicAdd(&listed_n, 1u);
                        if (at < LIST) list[at] = word(u, e);
                    }
        }
        __syncthreads();
        int n = (int)listed_n;
        if (n > LIST) { // many logits equal to the bound: only those above it, then as many equal ones as are missing, in order
            __syncthreads();
            if (tid == 0) listed_n = 0u;
            __syncthreads();
            if (lane_max > bv) {
#pragma unroll
                for (int u = 0; u < NL; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (v[u][e] > bv) list[atomicAdd(&listed_n, 1u)] = word(u, e);
            }
            __syncthreads();
            n = (int)listed_n;
            const int above = n;
            for (int u = 0; u < NL && n < k; ++u) { // n is the same in every thread
                int mine = 0;
                half8_t vu = v[0];
#pragma unroll
                for (int w = 1; w < NL; ++w) vu = w == u ? v[w] : vu;
#pragma unroll
                for (int e = 0; e < 8; ++e) mine += vu[e] == bv;
                int before = mine; // inclusive over the wavefront's lanes
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int q = __shfl_up(before, o);
                    if (lane >= o) before += q;
                }
                if (lane == 63) red[wave] = (uint32_t)before;
                __syncthreads();
                int at = n + before - mine, total = 0;
                for (int w = 0; w < LP_WAVES; ++w) {
                    if (w < wave) at += (int)red[w];
                    total += (int)red[w];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (vu[e] == bv) {
                        if (at < k) list[at] = bound << 16 | (uint32_t)(0xffff - ((u * LP_THREADS + tid) * 8 + e));
                        ++at;
                    }
                n += total;
                __syncthreads();
            }
            if (above < k && n > k) n = k;
        }
        lp_rank(list, n, k, best, red);
    }
    // ---- 4. several chunks: leave this one's result; the row's last workgroup goes on -------------------------------------
    if (a.chunks > 1) {
        // Handed over by device-scope stores (written through to where every XCD reads them) that are complete before the
        // counter moves, and device-scope loads: a fence in each of thousands of workgroups would write the L2 back each time
        // (2048 rows: 3640 us with fences).
        const size_t at = row * a.chunks + chunk;
        if (tid < 3) lp_put(a.stats + at * 4 + tid, __builtin_bit_cast(uint32_t, tid == 0 ? st.m : tid == 1 ? st.s : st.t));
        if (tid < k) lp_put(a.listed + at * k + tid, best[tid]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) is_last = __hip_atomic_fetch_add(a.counters + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1;
        __syncthreads();
        if (!is_last) return;
        if (tid == 0) a.counters[row] = 0; // ready for the next launch
        float mine[3] = {-INFINITY, 0.f, 0.f};
        if (lane < a.chunks)
#pragma unroll
            for (int i = 0; i < 3; ++i) mine[i] = __builtin_bit_cast(float, lp_get(a.stats + (row * a.chunks + lane) * 4 + i));
        M = wave_max(mine[0]);
        const LpStats p = lp_rebase({mine[0], mine[1], mine[2]}, M, c);
        st = {M, wave_sum(p.s), wave_sum(p.t)};
        if (k > 0) {
            // the chunks' lists as one, in the order of the row; the same bound as above
            const uint32_t *listed = a.listed + row * a.chunks * k;
            const int total = a.chunks * k;
            uint32_t w[LP_MERGE], lane_best = 0u;
#pragma unroll
            for (int j = 0; j < LP_MERGE; ++j) {
                const int q = tid + LP_THREADS * j;
                const uint32_t e = q < total ? lp_get(listed + q) : 0u;
                w[j] = e ? (e & 0xffff0000u) | (uint32_t)(0xffff - q) : 0u;
                lane_best = w[j] > lane_best ? w[j] : lane_best;
            }
            const uint32_t bound_w = lp_kth_key(lane_best >> 16, k);
            if (lane == 0) red[wave] = bound_w;
            if (tid == 0) listed_n = 0u;
            __syncthreads();
            uint32_t bound = LP_LOWEST;
#pragma unroll
            for (int i = 0; i < LP_WAVES; ++i) bound = red[i] > bound ? red[i] : bound;
#pragma unroll
            for (int j = 0; j < LP_MERGE; ++j)
                if (w[j] >> 16 >= bound) list[atomicAdd(&listed_n, 1u)] = w[j];
            __syncthreads();
            lp_rank(list, (int)listed_n, k, best, red);
            if (tid < k && best[tid]) { // back to the place in the row
                const int q = 0xffff - (int)(best[tid] & 0xffffu);
                list[tid] = (uint32_t)(q / k * CHUNK) + 0xffffu - (lp_get(listed + q) & 0xffffu);
            }
        }
    } else if (tid < k) {
        list[tid] = 0xffffu - (best[tid] & 0xffffu);
    }
    // ---- 5. results ------------------------------------------------------------------------------------------------------
    const bool invalid = st.s != st.s, none = st.s == 0.f;
    const float m0 = none ? 0.f : st.m, log_s = none ? 0.f : logf(st.s);
    if (tid == 0) a.entropy[row] = invalid ? NAN : none ? 0.f : log_s - st.t / st.s * 0.693147180559945309f;
    if (tid < a.n_ids) {
        const int id = a.ids[row * a.n_ids + tid];
        float lp = NAN;
        if (id >= 0 && id < a.vocab && !invalid) lp = ((float)x[id] - m0) * a.inv_t - log_s;
        a.logprob[row * a.n_ids + tid] = lp;
    }
    if (tid < k) {
        const bool some = best[tid] != 0u && !invalid;
        a.top_ids[row * k + tid] = some ? (int)list[tid] : -1;
        a.top[row * k + tid] = invalid ? NAN : some ? ((float)lp_value(best[tid] >> 16) - m0) * a.inv_t - log_s : -INFINITY;
    }
}

// Loads per thread of a chunk.  Few rows are cut finely, so that their logits come from many compute units at once (at most
// LP_MAX_CHUNKS pieces); many rows coarsely, so that less is joined.
static int lp_loads(int rows, int vocab) {
    int nl = 1;
    while (nl < LP_MAX_LOADS) {
        const int one = LP_THREADS * 8 * nl, chunks = (vocab + one - 1) / one, coarser = (vocab + 2 * one - 1) / (2 * one);
        if (chunks <= LP_MAX_CHUNKS && (chunks == 1 || (long long)rows * coarser < 512)) break;
        nl *= 2;
    }
    return nl;
}
static int lp_chunks(int rows, int vocab) {
    const int one = LP_THREADS * 8 * lp_loads(rows, vocab);
    return (vocab + one - 1) / one;
}

template <int NL> static void lp_launch(const LpArgs &a, int rows, hipStream_t s) {
    logprobs_kernel<NL><<<dim3(a.chunks, rows), dim3(LP_THREADS), 0, s>>>(a);
}

extern "C" {

// counters of LP_SLICE rows, then the statistics and lists of one launch
size_t llm_logprobs_workspace_bytes(int rows, int vocab, int k) {
    if (rows < 1 || vocab < 1 || vocab > LP_MAX_VOCAB || k < 0) return sizeof(int) * LP_SLICE;
    const size_t n = (size_t)(rows < LP_SLICE ? rows : LP_SLICE) * lp_chunks(rows, vocab);
    return sizeof(int) * LP_SLICE + n * sizeof(uint32_t) * (4 + k);
}

int llm_logprobs(const uint16_t *logits, int ld, int rows, int vocab, float temperature, const int32_t *ids, int n_ids,
                 float *logprob, float *entropy, int k, int32_t *top_ids, float *top_logprob, void *workspace, llm_stream_t stream) {
    LLM_REQUIRE(rows >= 0 && vocab >= 1 && ld >= vocab, "llm_logprobs: %d rows of %d logits, ld=%d", rows, vocab, ld);
    LLM_REQUIRE(vocab <= LP_MAX_VOCAB, "llm_logprobs: %d logits per row (at most %d)", vocab, LP_MAX_VOCAB);
    LLM_REQUIRE(temperature >= FLT_MIN && temperature <= FLT_MAX, "llm_logprobs: temperature %g", (double)temperature);
    LLM_REQUIRE(n_ids >= 0 && n_ids <= LP_MAX_IDS, "llm_logprobs: %d given tokens per row (0..%d)", n_ids, LP_MAX_IDS);
    LLM_REQUIRE(k >= 0 && k <= LP_MAX_TOP && k <= vocab, "llm_logprobs: top %d of %d (at most %d)", k, vocab, LP_MAX_TOP);
    LLM_REQUIRE(logits && entropy && workspace && (n_ids == 0 || (ids && logprob)) && (k == 0 || (top_ids && top_logprob)),
                "llm_logprobs: null pointer");
    LLM_REQUIRE(((uintptr_t)logits & 1u) == 0 && aligned16(workspace) &&
                    (((uintptr_t)ids | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_logprob) & 3u) == 0,
                "llm_logprobs: logits must be aligned to 2 bytes, the workspace to 16, the others to 4");
    LpArgs a = {};
    a.ld = (size_t)ld;
    a.vocab = vocab;
    a.n_ids = n_ids;
    a.k = k;
    a.chunks = lp_chunks(rows, vocab);
    a.inv_t = 1.f / temperature;
    a.counters = (int *)workspace;
    a.stats = (uint32_t *)workspace + LP_SLICE;
    hipStream_t s = (hipStream_t)stream;
    for (int r0 = 0; r0 < rows; r0 += LP_SLICE) {
        const int n = rows - r0 < LP_SLICE ? rows - r0 : LP_SLICE;
        a.listed = a.stats + (size_t)n * a.chunks * 4;
        a.x = (const half_t *)logits + (size_t)r0 * ld;
        a.ids = ids + (size_t)r0 * n_ids;
        a.logprob = logprob + (size_t)r0 * n_ids;
        a.entropy = entropy + r0;
        a.top_ids = top_ids + (size_t)r0 * k;
        a.top = top_logprob + (size_t)r0 * k;
        switch (lp_loads(rows, vocab)) {
        case 1: lp_launch<1>(a, n, s); break;
        case 2: lp_launch<2>(a, n, s); break;
        case 4: lp_launch<4>(a, n, s); break;
        default: lp_launch<8>(a, n, s); break;
        }
        LLM_LAUNCH_CHECK("logprobs_kernel");
    }
    return LLM_OK;
}

} // extern "C"
