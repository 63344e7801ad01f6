// Log probabilities of given tokens, entropy and the best alternatives of rows of fp16 logits.
//
//   y = x / temperature, m = max y, S = sum exp(y - m)
//   logprob(i) = (y_i - m) - ln S,   entropy = ln S - sum (y - m) exp(y - m) / S
//
// One pass over the logits.  A row is cut into chunks, one workgroup each; its wavefronts go through the chunk's segments on
// their own, the next segment's loads in flight while one is worked on, and meet at the end of the chunk only; the workgroup of
// a row that finishes last joins the chunks.
//
// What bounds it: many rows, the logits' bytes (read once): 2048 rows of 128256, the best alternative and one given token 96 us,
// 5.5 TB/s (a large copy reads and writes 5.07); the 20 best 125 us, what listing candidates and cutting the lists adds to the six
// operations a logit.  Few rows, the kernel's latency: 16 rows, 5 best, 8.5 us, one row, 20 best, 10.2 us a call (10.6 on the chip), of
// which 4.7 are the row without alternatives and 6 the two levels of lists; a chunk of 2048 alone takes 2.2 and, with 20, 5.2.
//
// Sums: exponentials are base 2, 2^((x - m) c) with c = log2(e) / temperature for the largest logit m so far.  The difference comes
// first: it is exact or rounded once, so the largest logit has weight 1 at any temperature (a fused x c - m c is off by the rounding
// of m c, which passes the range of 2^y at m / temperature = 4e9).  A larger m rescales the lane's sums.
//
// The k best (k <= 32) without a sort: the k-th largest of a wavefront's 64 running lane maxima is a lower bound of its k-th
// largest logit, found digit by digit on 16-bit order keys (ballots and bit counts, two bits a step).  The few logits from there up are
// appended to the wavefront's list in LDS; a list that would overflow (many equal logits, rising rows) is cut down to its k
// best, after which only larger logits can enter, since equal ones further back lose.  A listed logit is a 64-bit word, order
// key above the complement of its index.
#include <cfloat>
#include <climits>
#include <cmath>

#include "common.hpp"

#define LP_THREADS 256
#define LP_WAVES (LP_THREADS / 64)
#define LP_MAX_TOP LLM_LOGPROBS_MAX_TOP
#define LP_MAX_IDS LLM_LOGPROBS_MAX_IDS
#define LP_MAX_CHUNKS 64       // of a row: one lane each when they are joined
#define LP_MAX_VOCAB (1 << 20)
#define LP_SLICE 4096          // rows per launch: a counter each at the front of the workspace
#define LP_WORKGROUPS 512      // aimed at
#define LP_LINE 32             // ints from one row's counter to the next: device-scope additions to one line wait for one another
#define LP_LIST 768            // words of a wavefront's list: a row of 16-byte loads (512 logits) behind what it holds
// Lanes above the bound up to which it stays, rather than being found anew.  With 0, 3, 8 and 16: 256 rows of 128256, 5 best, 27.1
// 26.1 28.7 30.8 us, 2048 rows 106.5 106.9 115.6 123.9; 20 best, 700 rows, 59.8 57.8 58.9 63.6.
#define LP_FEW 3
#define LP_JOIN (LP_MAX_CHUNKS * LP_MAX_TOP / LP_THREADS) // listed logits per thread when chunks are joined
#define LP_LOWEST 0x0400u      // order key of -65504, the lowest logit that has a probability

typedef unsigned long long lp_word;
typedef unsigned long long lp_pair __attribute__((ext_vector_type(2)));

struct LpArgs {
    const half_t *x;
    size_t ld;
    int vocab, n_ids, k, chunks, chunk_len;
    float inv_t;
    const int32_t *ids;
    float *logprob, *entropy, *top;
    int32_t *top_ids;
    int *counters;
    lp_word *listed;    // [row][chunk][k]
    uint32_t *stats;    // [row][chunk][4]: m, S, sum y 2^y as bits
};

struct LpStats {
    float m, s, t; // largest logit, sum of 2^(d c), sum of d 2^(d c) with d = x - m
};

__device__ __forceinline__ void lp_put(uint32_t *p, uint32_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint32_t lp_get(const uint32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void lp_put(lp_word *p, lp_word v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ lp_word lp_get(const lp_word *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

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
__device__ __forceinline__ lp_word lp_make(half_t h, int index) { return (lp_word)lp_key(h) << 32 | (uint32_t)~index; }
__device__ __forceinline__ uint32_t lp_word_key(lp_word w) { return (uint32_t)(w >> 32); }

__device__ __forceinline__ float lp_base(float m) { return m == -INFINITY ? 0.f : m; }

// sums relative to the reference of a larger maximum M
__device__ __forceinline__ LpStats lp_rebase(LpStats p, float M, float c) {
    const float d = lp_base(p.m) - lp_base(M), f = p.s == 0.f ? 0.f : __builtin_amdgcn_exp2f(d * c);
    return {M, f * p.s, f == 0.f ? 0.f : f * (p.t + d * p.s)};
}

// k-th largest of the lanes' keys (0: fewer than k lanes have one); two bits at a time, the three counts of a step side by side
__device__ __forceinline__ uint32_t lp_kth_key(uint32_t key, int k) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 14; bit >= 0; bit -= 2) {
        const int c1 = __popcll(__builtin_amdgcn_ballot_w64(key >= (t | 1u << bit)));
        const int c2 = __popcll(__builtin_amdgcn_ballot_w64(key >= (t | 2u << bit)));
        const int c3 = __popcll(__builtin_amdgcn_ballot_w64(key >= (t | 3u << bit)));
        t |= (c3 >= k ? 3u : c2 >= k ? 2u : c1 >= k ? 1u : 0u) << bit;
    }
    return t;
}

// LDS written by some lanes of a wavefront, read by others: its operations are carried out in order, the compiler keeps theirs
__device__ __forceinline__ void lp_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Appends the words of the lanes in `who` (mine: this lane is one) to the wavefront's list of n words; returns the new length.
__device__ __forceinline__ int lp_append(lp_word *list, int n, unsigned long long who, bool mine, lp_word w) {
    const int before = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
    if (mine) list[n + before] = w;
    return n + __popcll(who);
}

// How many of list[0 .. n8) are above w: n8 is a multiple of eight (zeros fill the list up), eight words in flight.
__device__ __forceinline__ int lp_rank(const lp_word *list, int n8, lp_word w) {
    int rank = 0;
    for (int j = 0; j < n8; j += 8) {
        lp_pair x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const lp_pair *>(list + j + 2 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) rank += (x[i][0] > w) + (x[i][1] > w);
    }
    return rank;
}

// The k largest of a wavefront's n <= LP_LIST distinct words to the front of its list, largest first, zeros behind them
// up to LP_MAX_TOP words.
__device__ __forceinline__ void lp_cut(lp_word *list, int n, int k) {
    const int lane = threadIdx.x % 64;
    lp_word w[LP_LIST / 64];
    auto spread = [&]() __attribute__((always_inline)) { // the list over the lanes
        lp_wave_sync();
        lp_word top = 0ull;
#pragma unroll
        for (int i = 0; i < LP_LIST / 64; ++i) {
            w[i] = lane + 64 * i < n ? list[lane + 64 * i] : 0ull;
            top = w[i] > top ? w[i] : top;
        }
        lp_wave_sync();
        return top;
    };
    if (n > 64) { // only what is not below the k-th largest of the lanes' largest: little more than k words, but for equal logits
        const uint32_t from = lp_kth_key(lp_word_key(spread()), k);
        n = 0;
#pragma unroll
        for (int i = 0; i < LP_LIST / 64; ++i) {
            const bool mine = w[i] != 0ull && lp_word_key(w[i]) >= from;
            const unsigned long long who = __builtin_amdgcn_ballot_w64(mine);
            if (who) n = lp_append(list, n, who, mine, w[i]);
        }
    }
    if (n <= 128) {
        if (lane < 8) list[n + lane] = 0ull;
        lp_wave_sync();
        const int n8 = (n + 7) & ~7;
        const lp_word a = lane < n ? list[lane] : 0ull, b = lane + 64 < n ? list[lane + 64] : 0ull;
        const int ra = lp_rank(list, n8, a), rb = n > 64 ? lp_rank(list, n8, b) : 0;
        lp_wave_sync();
        if (a && ra < k) list[ra] = a;
        if (b && rb < k) list[rb] = b;
    } else { // their maximum, k times
        lp_word top = spread();
        for (int r = 0; r < k; ++r) {
            for (int o = 32; o; o >>= 1) {
                const lp_word q = __shfl_xor(top, o);
                top = q > top ? q : top;
            }
            if (lane == 0) list[r] = top;
            lp_word rest = 0ull;
#pragma unroll
            for (int i = 0; i < LP_LIST / 64; ++i) {
                w[i] = w[i] == top ? 0ull : w[i];
                rest = w[i] > rest ? w[i] : rest;
            }
            top = rest;
        }
    }
    if (lane >= (n < k ? n : k) && lane < LP_MAX_TOP) list[lane] = 0ull;
    lp_wave_sync();
}

// A wavefront's list made ready for lp_join_waves: cut unless it is hardly longer than k (joining costs every word of it four times
// what cutting does), and a multiple of eight with zeros.  Returns its length, at most 64.
__device__ __forceinline__ int lp_ready(lp_word *list, int n, int k) {
    if (n > k + 8) {
        lp_cut(list, n, k);
        n = k; // zeros in the place of what is missing
    }
    const int lane = threadIdx.x % 64, n8 = (n + 7) & ~7;
    if (lane < n8 - n) list[n + lane] = 0ull;
    return n8;
}

// The wavefronts' lists (n8[w] words each) into best, largest first.  All threads call it, behind a barrier.
__device__ __forceinline__ void lp_join_waves(const lp_word *lists, const int *n8, int k, lp_word *best) {
    static_assert(LP_MAX_TOP + 8 <= 64, "a word per thread");
    const int tid = threadIdx.x;
    int size[LP_WAVES], from = 0; // the first threads take a word each
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w) size[w] = n8[w];
    if (tid < k) best[tid] = 0ull;
    __syncthreads();
    int at = -1;
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w) {
        if (tid >= from && tid < from + size[w]) at = w * LP_LIST + tid - from;
        from += size[w];
    }
    if (at >= 0) {
        const lp_word mine = lists[at];
        int rank = 0;
#pragma unroll
        for (int w = 0; w < LP_WAVES; ++w) rank += lp_rank(lists + w * LP_LIST, size[w], mine);
        if (mine && rank < k) best[rank] = mine;
    }
    __syncthreads();
}

// NL 16-byte loads per lane and segment.
template <int NL>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const LpArgs a) {
    constexpr int SEG = 64 * 8 * NL;
    extern __shared__ __attribute__((aligned(16))) lp_word lists[]; // LP_WAVES lists of LP_LIST words when k > 0
    __shared__ lp_word best[LP_MAX_TOP];
    __shared__ float part[LP_WAVES][3];
    __shared__ int is_last, ready[LP_WAVES];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, chunk = blockIdx.x, k = a.k;
    const size_t row = blockIdx.y;
    const half_t *x = a.x + row * a.ld;
    const float c = a.inv_t * 1.44269504088896341f;
    float one = 1.f;
    asm("" : "+v"(one)); // not folded: a multiplication, so that conversion and difference are one instruction
    const half_t ninf = __builtin_bit_cast(half_t, (uint16_t)0xfc00u);
    lp_word *list = lists + wave * LP_LIST;

    // the given tokens' logits, asked for in front of everything else (only the workgroup that ends the row uses them)
    int id = -1;
    half_t given = ninf;
    if (tid < a.n_ids) {
        id = a.ids[row * a.n_ids + tid];
        if (id >= 0 && id < a.vocab) given = x[id];
    }
    // ---- 1. the wavefront's segments: wave, wave + LP_WAVES, ... of the chunk ---------------------------------------------
    const int begin = chunk * a.chunk_len, end = begin + a.chunk_len < a.vocab ? begin + a.chunk_len : a.vocab;
    LpStats st = {-INFINITY, 0.f, 0.f}; // m of the wavefront, sums of the lane
    half_t lane_best = ninf;
    uint32_t bound = LP_LOWEST; // order key from which on a logit is listed, and its value
    half_t from = lp_value(bound);
    int n = 0;
    half8_t v[NL], next[NL];
    auto load = [&](half8_t (&d)[NL], int s0) __attribute__((always_inline)) {
        if (s0 + SEG <= end) {
#pragma unroll
            for (int u = 0; u < NL; ++u) d[u] = lp_load8(x + s0 + (u * 64 + lane) * 8);
            return;
        }
#pragma unroll
        for (int u = 0; u < NL; ++u) { // the chunk's last segment: -inf behind the end
            const int i = s0 + (u * 64 + lane) * 8;
            d[u] = half8_t{ninf, ninf, ninf, ninf, ninf, ninf, ninf, ninf};
            if (i + 8 <= end) d[u] = lp_load8(x + i);
            else if (i < end)
                for (int e = 0; e < 8; ++e) d[u][e] = i + e < end ? x[i + e] : ninf;
        }
    };
    int s0 = begin + wave * SEG;
    if (s0 < end) load(v, s0);
    for (; s0 < end; s0 += LP_WAVES * SEG) {
        const bool more = s0 + LP_WAVES * SEG < end;
        if (more) load(next, s0 + LP_WAVES * SEG);
        half_t lane_max[NL], top = ninf; // a NaN loses against any number here; the sums find it
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            const half4_t m4 = __builtin_elementwise_max(__builtin_shufflevector(v[u], v[u], 0, 1, 2, 3), __builtin_shufflevector(v[u], v[u], 4, 5, 6, 7));
            const half2_t m2 = __builtin_elementwise_max(__builtin_shufflevector(m4, m4, 0, 1), __builtin_shufflevector(m4, m4, 2, 3));
            lane_max[u] = m2[0] > m2[1] || m2[1] != m2[1] ? m2[0] : m2[1];
            top = lane_max[u] > top ? lane_max[u] : top;
        }
        if (__builtin_amdgcn_ballot_w64((float)top > st.m)) st = lp_rebase(st, fmaxf(st.m, wave_max((float)top)), c);
        const float base = lp_base(st.m);
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            float p[8], t = 0.f; // eight at a time: a lane's sums take an eighth of the roundings one after the other
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = fmaf((float)v[u][e], one, -base);
                p[e] = __builtin_amdgcn_exp2f(d * c);
                t = fmaf(fmaxf(d, -FLT_MAX), p[e], t); // -inf times zero is zero here; a NaN is in p already
            }
            st.s += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            st.t += t;
        }
        lane_best = top > lane_best ? top : lane_best;
        const int lanes = k > 0 ? __popcll(__builtin_amdgcn_ballot_w64(top >= from)) : 0;
        if (lanes) {
            if (k == 1 || lanes > LP_FEW) { // the lanes' maxima have moved enough for the bound to follow
                const uint32_t kth = k == 1 ? lp_key((half_t)st.m) : lp_kth_key(lane_best == ninf ? 0u : lp_key(lane_best), k);
                bound = kth > bound ? kth : bound;
                from = lp_value(bound);
            }
            uint32_t some = 0u; // loads with a logit from the bound on
#pragma unroll
            for (int u = 0; u < NL; ++u) some |= __builtin_amdgcn_ballot_w64(lane_max[u] >= from) ? 1u << u : 0u;
            for (int u = 0; some; ++u, some >>= 1) {
                if (!(some & 1u)) continue;
                if (n > LP_LIST - 512) {
                    lp_cut(list, n, k);
                    n = k;
                    const uint32_t above = lp_word_key(list[k - 1]) + 1u; // an equal logit further back is not among the k best
                    bound = above > bound ? above : bound;
                    from = lp_value(bound);
                }
                half8_t w = v[0];
#pragma unroll
                for (int i = 1; i < NL; ++i) w = i == u ? v[i] : w;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned long long who = __builtin_amdgcn_ballot_w64(w[e] >= from);
                    if (who) n = lp_append(list, n, who, w[e] >= from, lp_make(w[e], s0 + (u * 64 + lane) * 8 + e));
                }
            }
        }
        if (more)
#pragma unroll
            for (int u = 0; u < NL; ++u) v[u] = next[u];
    }
    // ---- 2. the workgroup's wavefronts -------------------------------------------------------------------------------------
    st.s = wave_sum(st.s);
    st.t = wave_sum(st.t);
    if (lane == 0) {
        part[wave][0] = st.m;
        part[wave][1] = st.s;
        part[wave][2] = st.t;
    }
    if (k > 0) {
        const int n8 = lp_ready(list, n, k);
        if (lane == 0) ready[wave] = n8;
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
    if (k > 0) lp_join_waves(lists, ready, k, best);
    // ---- 3. several chunks: leave this one's result; the row's last workgroup goes on -------------------------------------
    if (a.chunks > 1) {
        // Handed over by device-scope stores (written through to where every XCD reads them) that are complete before the
        // counter moves, and device-scope loads: a fence in each of thousands of workgroups would write the L2 back each time
        // (2048 rows: 3640 us with fences).
        const size_t at = row * a.chunks + chunk;
        if (tid < 3) lp_put(a.stats + at * 4 + tid, __builtin_bit_cast(uint32_t, tid == 0 ? st.m : tid == 1 ? st.s : st.t));
        if (tid < k) lp_put(a.listed + at * k + tid, best[tid]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) is_last = __hip_atomic_fetch_add(a.counters + row * LP_LINE, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1;
        __syncthreads();
        if (!is_last) return;
        if (tid == 0) a.counters[row * LP_LINE] = 0; // ready for the next launch
        lp_word w[LP_JOIN]; // all of what the chunks left is asked for at once
        const lp_word *listed = a.listed + row * a.chunks * k;
#pragma unroll
        for (int j = 0; j < LP_JOIN; ++j) {
            const int q = tid + LP_THREADS * j;
            w[j] = q < a.chunks * k ? lp_get(listed + q) : 0ull;
        }
        float mine[3] = {-INFINITY, 0.f, 0.f};
        if (lane < a.chunks)
#pragma unroll
            for (int i = 0; i < 3; ++i) mine[i] = __builtin_bit_cast(float, lp_get(a.stats + (row * a.chunks + lane) * 4 + i));
        M = wave_max(mine[0]);
        const LpStats p = lp_rebase({mine[0], mine[1], mine[2]}, M, c);
        st = {M, wave_sum(p.s), wave_sum(p.t)};
        if (k > 0) {
            lp_word top = 0ull;
#pragma unroll
            for (int j = 0; j < LP_JOIN; ++j) top = w[j] > top ? w[j] : top;
            const uint32_t kth = lp_kth_key(lp_word_key(top), k); // the same bound, on what the chunks listed
            n = 0;
#pragma unroll
            for (int j = 0; j < LP_JOIN; ++j) {
                const bool mine_too = w[j] != 0ull && lp_word_key(w[j]) >= kth;
                const unsigned long long who = __builtin_amdgcn_ballot_w64(mine_too);
                if (who) n = lp_append(list, n, who, mine_too, w[j]);
            }
            const int n8 = lp_ready(list, n, k);
            if (lane == 0) ready[wave] = n8;
            __syncthreads();
            lp_join_waves(lists, ready, k, best);
        }
    }
    // ---- 4. results ------------------------------------------------------------------------------------------------------
    const bool invalid = st.s != st.s, none = st.s == 0.f;
    const float m0 = none ? 0.f : st.m, mean = none ? 0.f : st.t / st.s * a.inv_t, log_s = none ? 0.f : logf(st.s);
    if (tid == 0) a.entropy[row] = invalid ? NAN : fmaxf(log_s - mean, 0.f); // where it is about 0, roundings may have either sign
    if (tid < a.n_ids) {
        float lp = NAN;
        if (id >= 0 && id < a.vocab && !invalid) lp = ((float)given - m0) * a.inv_t - log_s;
        a.logprob[row * a.n_ids + tid] = lp;
    }
    if (tid < k) {
        const bool some = best[tid] != 0ull && !invalid;
        a.top_ids[row * k + tid] = some ? (int)~(uint32_t)best[tid] : -1;
        a.top[row * k + tid] = invalid ? NAN : some ? ((float)lp_value(lp_word_key(best[tid])) - m0) * a.inv_t - log_s : -INFINITY;
    }
}

// How a row is cut.  Few rows: finely, so that their logits come from many compute units at once, but into LP_MAX_CHUNKS pieces
// at most; many rows: coarsely, so that less is joined.  Aimed at LP_WORKGROUPS; with 256, 512 and 1024, rows of 128256: 64 rows,
// 20 best, 21.0 17.8 15.9 us, 256 rows, 5 best, 30.1 26.1 24.8, but 700 rows, 20 best, 58 58 69.
// Short chunks in short segments, so that all wavefronts have one, long chunks in long ones with more loads in flight: with 1, 2
// and 4 loads per lane 16 rows (chunks of 4096), 5 best, 9.5 8.5 8.9 us, one row (2048), 20 best, 10.2 and, with 4, 11.8, 2048 whole
// rows, 5 best, 115 with one and 107 with 4.
struct LpCut {
    int nl, chunk_len, chunks;
};
static LpCut lp_cut_row(int rows, int vocab) {
    int want = (LP_WORKGROUPS + rows - 1) / rows;
    if (want > LP_MAX_CHUNKS) want = LP_MAX_CHUNKS;
    int len = (vocab + want - 1) / want;
    LpCut r = {};
    r.nl = len <= 2048 ? 1 : len <= 4096 ? 2 : 4;
    const int unit = LP_THREADS * 8 * r.nl;
    r.chunk_len = (len + unit - 1) / unit * unit;
    r.chunks = (vocab + r.chunk_len - 1) / r.chunk_len;
    return r;
}

template <int NL> static void lp_launch(const LpArgs &a, int rows, hipStream_t s) {
    const size_t smem = a.k > 0 ? sizeof(lp_word) * LP_WAVES * LP_LIST : 0;
    logprobs_kernel<NL><<<dim3(a.chunks, rows), dim3(LP_THREADS), smem, s>>>(a);
}

extern "C" {

// Counters of LP_SLICE rows, then the statistics and lists of one launch.  Fewer rows are cut into more chunks each, so this is a
// bound for all calls of up to `rows` rows, whatever their vocabulary: rows * ceil(LP_WORKGROUPS / rows) < LP_WORKGROUPS + rows chunks.
size_t llm_logprobs_workspace_bytes(int rows, int vocab, int k) {
    if (rows < 1 || vocab < 1 || vocab > LP_MAX_VOCAB || k < 0) return sizeof(int) * LP_SLICE * LP_LINE;
    const size_t r = rows < LP_SLICE ? rows : LP_SLICE, most = r + LP_WORKGROUPS - 1, n = r * LP_MAX_CHUNKS < most ? r * LP_MAX_CHUNKS : most;
    return sizeof(int) * LP_SLICE * LP_LINE + n * (sizeof(uint32_t) * 4 + sizeof(lp_word) * k);
}

int llm_logprobs(const uint16_t *logits, int ld, int rows, int vocab, float temperature, const int32_t *ids, int n_ids,
                 float *logprob, float *entropy, int k, int32_t *top_ids, float *top_logprob, void *workspace, llm_stream_t stream) {
    LLM_REQUIRE(rows >= 0 && vocab >= 1 && ld >= vocab, "llm_logprobs: %d rows of %d logits, ld=%d", rows, vocab, ld);
    LLM_REQUIRE(rows <= INT_MAX - LP_SLICE, "llm_logprobs: %d rows (at most %d)", rows, INT_MAX - LP_SLICE);
    LLM_REQUIRE(vocab <= LP_MAX_VOCAB, "llm_logprobs: %d logits per row (at most %d)", vocab, LP_MAX_VOCAB);
    LLM_REQUIRE(temperature >= 1e-30f && temperature <= FLT_MAX, "llm_logprobs: temperature %g (at least 1e-30)", (double)temperature);
    LLM_REQUIRE(n_ids >= 0 && n_ids <= LP_MAX_IDS, "llm_logprobs: %d given tokens per row (0..%d)", n_ids, LP_MAX_IDS);
    LLM_REQUIRE(k >= 0 && k <= LP_MAX_TOP && k <= vocab, "llm_logprobs: top %d of %d (at most %d)", k, vocab, LP_MAX_TOP);
    LLM_REQUIRE(logits && entropy && workspace && (n_ids == 0 || (ids && logprob)) && (k == 0 || (top_ids && top_logprob)),
                "llm_logprobs: null pointer");
    LLM_REQUIRE(((uintptr_t)logits & 1u) == 0 && aligned16(workspace) &&
                    (((uintptr_t)ids | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_logprob) & 3u) == 0,
                "llm_logprobs: logits must be aligned to 2 bytes, the workspace to 16, the others to 4");
    if (rows == 0) return LLM_OK;
    LpArgs a = {};
    a.ld = (size_t)ld;
    a.vocab = vocab;
    a.n_ids = n_ids;
    a.k = k;
    const LpCut cut = lp_cut_row(rows, vocab);
    a.chunks = cut.chunks;
    a.chunk_len = cut.chunk_len;
    a.inv_t = 1.f / temperature;
    a.counters = (int *)workspace;
    a.stats = (uint32_t *)workspace + LP_SLICE * LP_LINE;
    hipStream_t s = (hipStream_t)stream;
    for (int r0 = 0; r0 < rows; r0 += LP_SLICE) {
        const int n = rows - r0 < LP_SLICE ? rows - r0 : LP_SLICE;
        a.listed = (lp_word *)(a.stats + (size_t)n * a.chunks * 4);
        a.x = (const half_t *)logits + (size_t)r0 * ld;
        a.ids = ids + (size_t)r0 * n_ids;
        a.logprob = logprob + (size_t)r0 * n_ids;
        a.entropy = entropy + r0;
        a.top_ids = top_ids + (size_t)r0 * k;
        a.top = top_logprob + (size_t)r0 * k;
        if (cut.nl == 1) lp_launch<1>(a, n, s);
        else if (cut.nl == 2) lp_launch<2>(a, n, s);
        else lp_launch<4>(a, n, s);
        LLM_LAUNCH_CHECK("logprobs_kernel");
    }
    return LLM_OK;
}

} // extern "C"
