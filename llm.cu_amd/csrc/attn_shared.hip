// Decode attention of a batch whose sequences share their first positions: one new token per sequence, RoPE and the
// cache append of that token folded in.
//
//   score(z, h, j) = q'(z, h) . K(j) / sqrt(hd),   out(z, h) = sum_j softmax_j(score) V(j)
//
// Positions 0..prefix_len-1 come from one prefix cache, positions prefix_len..p_z-1 from the sequence's own cache (row r
// holds position row0 + r), position p_z is the new token, whose rotated key and value are appended to the own cache.
#include <cfloat>
#include <cmath>

#include "common.hpp"

struct SharedArgs {
    const half_t *qkv;
    int ldq;
    half_t *out;
    int ldo;
    const float *table;
    int batch, n_kv_heads, max_pos, prefix_max;
    int max_prefix, max_tail; // bounds that the launch was sized for: what a descriptor holds beyond them is clamped
    // host form: everything by value; device form: the descriptor and element offsets into its caches
    const llm_shared_desc *desc;
    size_t prefix_offset, cache_offset;
    llm_shared_desc host;
};

// What one sequence reads and writes, inside the bounds of its caches whatever a descriptor holds.
struct SharedSeq {
    const half_t *kp, *vp; // prefix caches
    half_t *kc, *vc;       // own caches
    int prefix;            // positions in the prefix cache
    int first;             // own row of position `prefix`
    int tail;              // own rows in front of the new token
};

template <bool DEV> __device__ __forceinline__ SharedSeq shared_seq(const SharedArgs &a, int z) {
    const llm_shared_desc &d = DEV ? *a.desc : a.host;
    SharedSeq s;
    s.kp = reinterpret_cast<const half_t *>(d.k_prefix) + a.prefix_offset;
    s.vp = reinterpret_cast<const half_t *>(d.v_prefix) + a.prefix_offset;
    s.kc = reinterpret_cast<half_t *>(d.seq.k_cache[z]) + a.cache_offset;
    s.vc = reinterpret_cast<half_t *>(d.seq.v_cache[z]) + a.cache_offset;
    int prefix = d.prefix_len, row0 = d.row0, tail = d.seq.pos[z] - d.prefix_len;
    if (DEV) {
        prefix = prefix < 0 ? 0 : prefix > a.max_prefix ? a.max_prefix : prefix;
        row0 = row0 < 0 ? 0 : row0 > prefix ? prefix : row0;
        if (prefix - row0 > a.max_pos - 1) row0 = prefix - (a.max_pos - 1);
        const int most = a.max_tail < a.max_pos - 1 - (prefix - row0) ? a.max_tail : a.max_pos - 1 - (prefix - row0);
        tail = tail < 0 ? 0 : tail > most ? most : tail;
    }
    s.prefix = prefix;
    s.first = prefix - row0;
    s.tail = tail;
    return s;
}

// ---------------------------------------------------------------------------------------------------------------
// Parts.  A workgroup takes one KV head and one span of cache rows: of the prefix, for the queries of all sequences (batch * G
// rows in QT tiles of 32), or of one sequence's own rows, for its G queries.  It leaves, per query row, the reference maximum,
// the sum and the unnormalised P.V; attn_shared_merge_kernel joins the spans and adds the new token.
//
// The products are the transposed ones of the prompt pass: S^T = K . Q^T and O^T += V^T . P^T on v_mfma_f32_32x32x16_f16, so that
// a lane holds one query's column and the accumulators of the first product are the operand of the second: with the K rows of a
// 32-key chunk read in the order pi(m) (bits 2 and 3 of m swapped), accumulator e of lane (n, hb) is key 16 (e / 8) + 8 hb + e % 8.
//
// K and V^T tiles of SK keys travel straight into a ring of LDS stages (buffer_load ... lds); a lane fetches the 16-byte chunk
// that the bank swizzle assigns to its slot.  The four wavefronts of a workgroup are QT query tiles x KG groups of keys x DH
// parts of the output dims (DH = 2: both compute the scores, each half of the output).
// ---------------------------------------------------------------------------------------------------------------
#define AS_WAVES 4
#define AS_THREADS (64 * AS_WAVES)
#define AS_LDS_PTR(p) ((__attribute__((address_space(3))) void *)(p))

template <int HD, int QT> struct AsShape {
    static constexpr int KG = QT == 4 ? 1 : QT == 2 ? 2 : HD >= 64 ? 2 : 4;
    static constexpr int DH = AS_WAVES / (QT * KG);
    static constexpr int SK = HD >= 64 ? 64 : 128;       // keys per stage
    static constexpr int NCH = SK / 32 / KG;             // chunks of a stage per wavefront
    static constexpr int TILE = SK * HD;                 // halves of a K or V^T tile
    static constexpr int NS = HD >= 128 ? 2 : 4;         // stages of the ring
    static constexpr int DT = HD / 32 / DH;              // 32-dim tiles of the output per wavefront
    static_assert(QT * KG * DH == AS_WAVES && NCH >= 1 && DT >= 1, "roles of the wavefronts");
};
template <int HD> constexpr int as_lds_halves() { return AsShape<HD, 1>::NS * 2 * AsShape<HD, 1>::TILE; }

// Spans of a launch, the same for every KV head.
struct AsSpans {
    int span;          // keys, a multiple of 128
    int n_prefix;      // spans of the longest prefix the launch is sized for
    int n_tail;        // spans of the longest tail, per sequence
    float *acc, *ml;   // [prefix: kvh][span][batch * G], then [tails: z][kvh][span][G] rows of HD (acc) and 2 (ml) floats
};

// Rows of one span: chunks of eight rows from `begin` on, of which lo .. hi - 1 count.
struct AsRange {
    int begin, lo, hi;
};
__device__ __forceinline__ AsRange as_prefix_range(const SharedSeq &s, const AsSpans &sp, int i) {
    const int b = i * sp.span, e = b + sp.span;
    return {b, b, e < s.prefix ? e : s.prefix};
}
__device__ __forceinline__ AsRange as_tail_range(const SharedSeq &s, const AsSpans &sp, int i) {
    const int b = (s.first & ~7) + i * sp.span, e = b + sp.span, end = s.first + s.tail;
    return {b, b > s.first ? b : s.first, e < end ? e : end};
}

template <int HD, int QT, class QueryRow>
__device__ __forceinline__ void as_span(half_t *smem, const half_t *kbase, const half_t *vbase, const int max_pos, const AsRange r,
                                        const int rows, QueryRow query, float *acc, float *ml) {
    using S = AsShape<HD, QT>;
    constexpr int SK = S::SK, KG = S::KG, DH = S::DH, NS = S::NS, DT = S::DT, TILE = S::TILE;
    constexpr int NC = HD / 8, NCV = SK / 8;                     // 16-byte chunks per K row / V^T row of a tile
    constexpr int LPW = TILE * 2 / 1024 / AS_WAVES;              // loads per wavefront, stage and tile (1 KB each)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const int qt = wave % QT, kg = wave / QT % KG, dh = wave / (QT * KG);
    const int n = lane % 32, hb = lane / 32;
    const int stages = (r.hi - r.begin + SK - 1) / SK;

    // ---- loads: instruction i of a wavefront covers rows 4 i + wave, in units of the rows that 1 KB holds ----
    const __amdgpu_buffer_rsrc_t rs_k = __builtin_amdgcn_make_buffer_rsrc((void *)kbase, 0, max_pos * HD * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t rs_v = __builtin_amdgcn_make_buffer_rsrc((void *)vbase, 0, HD * max_pos * 2, 0x00020000);
    auto swz = [](int row, int chunks) { return row / (16 / chunks) & (chunks - 1); };
    const int krow = wave * (64 / NC) + lane / NC, vrow = wave * (64 / NCV) + lane / NCV;
    const int kchunk = lane % NC ^ swz(krow, NC), vchunk = lane % NCV ^ swz(vrow, NCV);
    const uint32_t koff = (uint32_t)krow * (HD * 2) + (uint32_t)kchunk * 16;
    const uint32_t voff = (uint32_t)vrow * (uint32_t)max_pos * 2u + (uint32_t)vchunk * 16;
    auto issue = [&](int slot, int st) __attribute__((always_inline)) { // stage st into slot % NS of the ring
        half_t *buf = smem + slot % NS * 2 * TILE;
        const int key = r.begin + st * SK;
        if (key + SK <= max_pos) {
#pragma unroll
            for (int i = 0; i < LPW; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_k, AS_LDS_PTR(buf + (i * AS_WAVES + wave) * 512), 16, koff,
                                                         (uint32_t)key * (HD * 2) + (uint32_t)i * (AS_WAVES * 1024), 0, 0);
#pragma unroll
            for (int i = 0; i < LPW; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_v, AS_LDS_PTR(buf + TILE + (i * AS_WAVES + wave) * 512), 16, voff,
                                                         (uint32_t)key * 2 + (uint32_t)i * (AS_WAVES * (64 / NCV)) * (uint32_t)max_pos * 2u, 0, 0);
            return;
        }
        // the tile reaches past the cache's last row: the rows behind it are read from the last ones (and masked later)
        const int vkey = key + 8 * vchunk < max_pos - 8 ? key + 8 * vchunk : max_pos - 8;
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
            const int row = key + i * AS_WAVES * (64 / NC) + krow;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_k, AS_LDS_PTR(buf + (i * AS_WAVES + wave) * 512), 16,
                                                     (uint32_t)(row < max_pos ? row : max_pos - 1) * (HD * 2) + (uint32_t)kchunk * 16, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < LPW; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_v, AS_LDS_PTR(buf + TILE + (i * AS_WAVES + wave) * 512), 16,
                                                     ((uint32_t)(i * AS_WAVES * (64 / NCV) + vrow) * (uint32_t)max_pos + (uint32_t)vkey) * 2u, 0, 0, 0);
    };

    // ---- queries: lane (n, hb) holds dims 16 ks + 8 hb .. + 7 of row 32 qt + n; rotated while the first tiles travel ----
    half8_t qf[HD / 16];
    float4_t cs[HD / 16][2];
    {
        const float *table;
        const half_t *q = query(32 * qt + n < rows ? 32 * qt + n : rows - 1, &table);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
            qf[ks] = load8(q + 16 * ks + 8 * hb);
            cs[ks][0] = *reinterpret_cast<const float4_t *>(table + 16 * ks + 8 * hb);
            cs[ks][1] = *reinterpret_cast<const float4_t *>(table + 16 * ks + 8 * hb + 4);
        }
    }
    // always NS stages (a short span's last one more than once): the number of loads in flight is known everywhere
    const int issued = stages > NS ? stages : NS;
#pragma unroll
    for (int st = 0; st < NS; ++st) issue(st, st < stages ? st : stages - 1);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = cs[ks][i / 4][i % 4];
        qf[ks] = rope_rotate8(qf[ks], c);
    }

    float16_t o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
    float m_run = -FLT_MAX, l_run = 0.f;
    const float c2 = 1.44269504088896341f / sqrtf((float)HD);
    const int pm = (n & ~0xC) | ((n & 8) >> 1) | ((n & 4) << 1); // pi(n)
    auto xhalf = [](float x, float &lo, float &hi) {
        auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        lo = __uint_as_float(w[0]);
        hi = __uint_as_float(w[1]);
    };

    for (int st = 0; st < stages; ++st) {
        // stage st has landed when at most the loads of the stages behind it are in flight
        const int behind = issued - 1 - st < NS - 1 ? issued - 1 - st : NS - 1;
        if (behind == 0) asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        else if (behind == 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LPW) : "memory");
        else if (behind == 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 * LPW) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(6 * LPW) : "memory");
        const half_t *ks_ = smem + st % NS * 2 * TILE, *vs_ = ks_ + TILE;
#pragma unroll
        for (int j = 0; j < S::NCH; ++j) {
            const int kc = 32 * (kg + KG * j), key0 = r.begin + st * SK + kc; // the chunk in the stage; its first key
            if (key0 >= r.hi || key0 + 32 <= r.lo) continue;                  // no key of the span (the same for every lane)
            const bool edge = key0 < r.lo || key0 + 32 > r.hi;
            float16_t s;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.f;
            const int krow_l = kc + pm;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(load8(ks_ + krow_l * HD + ((2 * ks + hb) ^ swz(krow_l, NC)) * 8), qf[ks], s, 0, 0, 0);
            if (edge) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = key0 + 16 * (e / 8) + 8 * hb + e % 8;
                    s[e] = key >= r.lo && key < r.hi ? s[e] : -FLT_MAX;
                }
            }
            // The reference of the exponentials moves when a score leaves it behind by 2^8: probabilities stay below 2^8 in
            // fp16 (their relative rounding does not depend on the reference), sums and output are fp32, and O^T is
            // rescaled a handful of times.
            float mx = -FLT_MAX, lo, hi;
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e]);
            xhalf(mx, lo, hi);
            mx = fmaxf(lo, hi) * c2;
            if (__builtin_amdgcn_ballot_w64(mx > m_run + 8.f)) {
                const float m_new = mx > m_run + 8.f ? mx : m_run, alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                l_run *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
                m_run = m_new;
            }
            // probabilities rounded to fp16, the operand type of the second product; their sum is that of the rounded ones, so
            // that numerator and denominator use the same weights
            half8_t p[2];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const half2_t h = {(half_t)__builtin_amdgcn_exp2f(fmaf(s[e], c2, -m_run)), (half_t)__builtin_amdgcn_exp2f(fmaf(s[e + 1], c2, -m_run))};
                p[e / 8][e % 8] = h[0];
                p[e / 8][e % 8 + 1] = h[1];
                l_run = __builtin_amdgcn_fdot2(h, half2_t{(half_t)1.f, (half_t)1.f}, l_run, false);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const int dim = 32 * (dh * DT + t) + n;
                    half8_t vf = load8(vs_ + dim * SK + ((kc / 8 + 2 * u + hb) ^ swz(dim, NCV)) * 8);
                    if (edge) { // rows outside the span may hold anything
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int key = key0 + 16 * u + 8 * hb + e;
                            vf[e] = key >= r.lo && key < r.hi ? vf[e] : (half_t)0.f;
                        }
                    }
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p[u], o[t], 0, 0, 0);
                }
            }
        }
        if (st + NS < stages) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); // every wavefront has read the stage
            issue(st, st + NS);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // a short span's spare loads
    {
        float lo, hi;
        xhalf(l_run, lo, hi);
        l_run = lo + hi;
    }
    // ---- the groups of keys into one (through the LDS of the ring), then out ----
    if (KG > 1) {
        constexpr int PER = 64 * (16 * DT + 2); // floats per wavefront
        float *ex = reinterpret_cast<float *>(smem);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int slot = qt + QT * dh;
        if (kg > 0) {
            float *d = ex + ((kg - 1) * QT * DH + slot) * PER;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) d[(16 * t + e) * 64 + lane] = o[t][e];
            d[16 * DT * 64 + lane] = m_run;
            d[(16 * DT + 1) * 64 + lane] = l_run;
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int g = 1; g < KG; ++g) {
            const float *d = ex + ((g - 1) * QT * DH + slot) * PER;
            const float m2 = d[16 * DT * 64 + lane], l2 = d[(16 * DT + 1) * 64 + lane];
            const float m_new = fmaxf(m_run, m2), f1 = __builtin_amdgcn_exp2f(m_run - m_new), f2 = __builtin_amdgcn_exp2f(m2 - m_new);
            l_run = l_run * f1 + l2 * f2;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[t][e] = o[t][e] * f1 + d[(16 * t + e) * 64 + lane] * f2;
            m_run = m_new;
        }
    }
    const int row = 32 * qt + n;
    if (row < rows) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4)
                *reinterpret_cast<float4_t *>(acc + (size_t)row * HD + 32 * (dh * DT + t) + 8 * e4 + 4 * hb) =
                    float4_t{o[t][4 * e4], o[t][4 * e4 + 1], o[t][4 * e4 + 2], o[t][4 * e4 + 3]};
        if (dh == 0 && hb == 0) {
            ml[2 * row] = m_run;
            ml[2 * row + 1] = l_run;
        }
    }
}

// Grid: (prefix spans, then tail spans of every sequence) x KV heads, the KV head fastest: consecutive workgroups go round the
// XCDs, so that a head's queries and tables stay in one XCD's L2.
template <int HD, int G, int QT, bool DEV>
__global__ __launch_bounds__(AS_THREADS, 2) void attn_shared_part_kernel(const SharedArgs a, const AsSpans sp) {
    extern __shared__ __attribute__((aligned(16))) half_t smem[];
    const int kvh = blockIdx.x % a.n_kv_heads, task = blockIdx.x / a.n_kv_heads;
    const int rows = a.batch * G;
    if (task < sp.n_prefix) {
        const SharedSeq s = shared_seq<DEV>(a, 0);
        const AsRange r = as_prefix_range(s, sp, task);
        if (r.lo >= r.hi) return;
        const size_t at = ((size_t)kvh * sp.n_prefix + task) * rows;
        auto query = [&](int row, const float **cs) {
            const int z = row / G;
            const SharedSeq sz = shared_seq<DEV>(a, z);
            *cs = a.table + (size_t)(sz.prefix + sz.tail) * HD;
            return a.qkv + (size_t)z * a.ldq + (size_t)(kvh * G + row % G) * HD;
        };
        as_span<HD, QT>(smem, s.kp + (size_t)kvh * a.prefix_max * HD, s.vp + (size_t)kvh * HD * a.prefix_max, a.prefix_max, r, rows, query,
                        sp.acc + at * HD, sp.ml + at * 2);
    } else {
        const int z = (task - sp.n_prefix) % a.batch, i = (task - sp.n_prefix) / a.batch;
        const SharedSeq s = shared_seq<DEV>(a, z);
        const AsRange r = as_tail_range(s, sp, i);
        if (r.lo >= r.hi) return;
        const size_t at = (size_t)a.n_kv_heads * sp.n_prefix * rows + (((size_t)z * a.n_kv_heads + kvh) * sp.n_tail + i) * G;
        auto query = [&](int row, const float **cs) {
            *cs = a.table + (size_t)(s.prefix + s.tail) * HD;
            return a.qkv + (size_t)z * a.ldq + (size_t)(kvh * G + row) * HD;
        };
        as_span<HD, 1>(smem, s.kc + (size_t)kvh * a.max_pos * HD, s.vc + (size_t)kvh * HD * a.max_pos, a.max_pos, r, G, query, sp.acc + at * HD,
                       sp.ml + at * 2);
    }
}

// One workgroup per query head and sequence: the new token's score, the spans' weights, the weighted sum; the first head of a
// group appends the new key and value.
#define AS_MERGE_THREADS 256
template <int HD, int G, bool DEV>
__global__ __launch_bounds__(AS_MERGE_THREADS) void attn_shared_merge_kernel(const SharedArgs a, const AsSpans sp) {
    constexpr int LPR = HD / 4, GROUPS = AS_MERGE_THREADS / LPR; // lanes per row of HD floats, rows side by side
    extern __shared__ float weight[]; // one per span
    __shared__ float l_all, w_new;
    __shared__ float4_t part[GROUPS][LPR];
    const int h = blockIdx.x, z = blockIdx.y, kvh = h / G, g = h % G, tid = threadIdx.x, lane = tid % 64;
    const int rows = a.batch * G, Hq = a.n_kv_heads * G;
    const SharedSeq s = shared_seq<DEV>(a, z);
    const int pos = s.prefix + s.tail, row = s.first + s.tail;
    const int np = (s.prefix + sp.span - 1) / sp.span, nt = s.tail > 0 ? ((s.first & 7) + s.tail + sp.span - 1) / sp.span : 0, ns = np + nt;
    const size_t pre = (size_t)kvh * sp.n_prefix * rows + (size_t)z * G + g;
    const size_t own = (size_t)a.n_kv_heads * sp.n_prefix * rows + ((size_t)z * a.n_kv_heads + kvh) * sp.n_tail * G + g;
    auto slot = [&](int i) { return i < np ? pre + (size_t)i * rows : own + (size_t)(i - np) * G; };
    const half_t *line = a.qkv + (size_t)z * a.ldq;
    const half_t *vn = line + (size_t)(Hq + a.n_kv_heads + kvh) * HD;
    if (tid < 64) {
        // the new token: eight dims per lane
        float dot = 0.f;
        if (lane < HD / 8) {
            const float *cs = a.table + (size_t)pos * HD + lane * 8;
            const half8_t q = rope_rotate8(load8(line + (size_t)h * HD + lane * 8), cs);
            const half8_t k = rope_rotate8(load8(line + (size_t)(Hq + kvh) * HD + lane * 8), cs);
            dot = dot8(q, k, 0.f);
            if (g == 0) {
                store8(s.kc + ((size_t)kvh * a.max_pos + row) * HD + lane * 8, k);
                const half8_t v = load8(vn + lane * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) s.vc[((size_t)kvh * HD + lane * 8 + e) * a.max_pos + row] = v[e];
            }
        }
        const float m_new = wave_sum(dot) * (1.44269504088896341f / sqrtf((float)HD));
        float M = m_new;
        for (int i = lane; i < ns; i += 64) {
            const float m = sp.ml[2 * slot(i)];
            weight[i] = m;
            M = fmaxf(M, m);
        }
        M = wave_max(M);
        float l = 0.f;
        for (int i = lane; i < ns; i += 64) {
            const float w = __builtin_amdgcn_exp2f(weight[i] - M);
            weight[i] = w;
            l += w * sp.ml[2 * slot(i) + 1];
        }
        l = wave_sum(l);
        if (lane == 0) {
            w_new = __builtin_amdgcn_exp2f(m_new - M);
            l_all = l + w_new;
        }
    }
    __syncthreads();
    const int d4 = tid % LPR, grp = tid / LPR;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int i = grp; i < ns; i += GROUPS) {
        const float4_t v = *reinterpret_cast<const float4_t *>(sp.acc + slot(i) * HD + 4 * d4);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += weight[i] * v[e];
    }
    part[grp][d4] = o;
    __syncthreads();
    if (tid < LPR) {
        const half4_t v = *reinterpret_cast<const half4_t *>(vn + 4 * d4);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = w_new * (float)v[e];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += part[i][d4][e];
        half_t *out = a.out + (size_t)z * a.ldo + (size_t)h * HD + 4 * d4;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = (half_t)(o[e] / l_all);
    }
}

// Spans per KV head, all sequences together: two workgroups on each of the 256 compute units, but enough for the prefix next to
// one span for each sequence's own rows.
static int as_target(int n_kv_heads, int batch) {
    const int fill = n_kv_heads < 512 ? 512 / n_kv_heads : 1;
    return fill > 2 * batch ? fill : 2 * batch;
}

static AsSpans as_spans(const SharedArgs &a) {
    AsSpans sp = {};
    const long long target = as_target(a.n_kv_heads, a.batch), total = a.max_prefix + (long long)a.batch * a.max_tail;
    for (long long span = (total / target + 127) / 128 * 128;; span += 128) {
        if (span == 0) continue;
        const long long np = (a.max_prefix + span - 1) / span, nt = a.max_tail > 0 ? (a.max_tail + 7 + span - 1) / span : 0;
        if (np + a.batch * nt <= target) { // holds at the latest where both are one
            sp.span = (int)span;
            sp.n_prefix = (int)np;
            sp.n_tail = (int)nt;
            return sp;
        }
    }
}

template <int HD, int G, int QT, bool DEV> static int launch_shared(const SharedArgs &a, AsSpans sp, hipStream_t s) {
    const size_t smem = sizeof(half_t) * as_lds_halves<HD>();
    auto kern = attn_shared_part_kernel<HD, G, QT, DEV>;
    static std::atomic<uint64_t> attr_done{0};
    if (smem > 48 * 1024) {
        int rc = llm_ensure_max_smem((const void *)kern, smem, attr_done);
        if (rc != LLM_OK) return rc;
    }
    const int tasks = sp.n_prefix + a.batch * sp.n_tail;
    if (tasks > 0) {
        kern<<<dim3((unsigned)tasks * a.n_kv_heads), dim3(AS_THREADS), smem, s>>>(a, sp);
        LLM_LAUNCH_CHECK("attn_shared_part_kernel");
    }
    attn_shared_merge_kernel<HD, G, DEV><<<dim3(a.n_kv_heads * G, a.batch), dim3(AS_MERGE_THREADS),
                                           sizeof(float) * (sp.n_prefix + sp.n_tail + 1), s>>>(a, sp);
    LLM_LAUNCH_CHECK("attn_shared_merge_kernel");
    return LLM_OK;
}

template <int HD, int G> static int launch_shared(const SharedArgs &a, void *ws, hipStream_t s) {
    AsSpans sp = as_spans(a);
    const int rows = a.batch * G;
    sp.acc = (float *)ws;
    sp.ml = sp.acc + ((size_t)a.n_kv_heads * sp.n_prefix * rows + (size_t)a.batch * a.n_kv_heads * sp.n_tail * G) * HD;
    constexpr int MAXR = G * LLM_MAX_BATCH;
    // as many query tiles as the batch fills
    if (rows <= 32 || MAXR <= 32) return a.desc ? launch_shared<HD, G, 1, true>(a, sp, s) : launch_shared<HD, G, 1, false>(a, sp, s);
    if (rows <= 64 || MAXR <= 64) return a.desc ? launch_shared<HD, G, MAXR >= 64 ? 2 : 1, true>(a, sp, s) : launch_shared<HD, G, MAXR >= 64 ? 2 : 1, false>(a, sp, s);
    return a.desc ? launch_shared<HD, G, MAXR >= 128 ? 4 : 1, true>(a, sp, s) : launch_shared<HD, G, MAXR >= 128 ? 4 : 1, false>(a, sp, s);
}

static int dispatch_shared(const char *name, const SharedArgs &a, int n_heads, int head_dim, void *ws, hipStream_t s) {
    const int G = n_heads / a.n_kv_heads;
#define AS_CASE(HD_, G_) \
    if (head_dim == HD_ && G == G_) return launch_shared<HD_, G_>(a, ws, s);
    AS_CASE(128, 4)
    AS_CASE(128, 8)
    AS_CASE(128, 1)
    AS_CASE(64, 4)
    AS_CASE(64, 1)
    AS_CASE(32, 4)
    AS_CASE(32, 1)
#undef AS_CASE
    llm_set_error("%s: head_dim=%d with group size %d is not built", name, head_dim, G);
    return LLM_ERR_INVALID;
}

static int shared_check(const char *name, const SharedArgs &a, int n_heads, int head_dim, const void *workspace) {
    LLM_REQUIRE(a.qkv && a.out && a.table && workspace, "%s: null pointer", name);
    LLM_REQUIRE(a.batch >= 1 && a.batch <= LLM_MAX_BATCH, "%s: batch=%d (1..%d)", name, a.batch, LLM_MAX_BATCH);
    LLM_REQUIRE(a.n_kv_heads > 0 && n_heads > 0 && n_heads % a.n_kv_heads == 0, "%s: heads %d/%d", name, n_heads, a.n_kv_heads);
    const int G = n_heads / a.n_kv_heads;
    const bool built = (head_dim == 128 && (G == 1 || G == 4 || G == 8)) || ((head_dim == 64 || head_dim == 32) && (G == 1 || G == 4));
    LLM_REQUIRE(built, "%s: head_dim=%d with group size %d is not built", name, head_dim, G);
    LLM_REQUIRE(a.max_pos > 0 && a.max_pos % 64 == 0 && a.prefix_max >= 0 && a.prefix_max % 64 == 0,
                "%s: max_pos=%d, prefix_max_pos=%d must be multiples of 64", name, a.max_pos, a.prefix_max);
    // one head's half of a cache is addressed with 32-bit byte offsets
    LLM_REQUIRE((size_t)a.max_pos * head_dim * sizeof(half_t) < (1ull << 31) && (size_t)a.prefix_max * head_dim * sizeof(half_t) < (1ull << 31),
                "%s: max_pos=%d, prefix_max_pos=%d: a head's keys must stay below 2 GiB", name, a.max_pos, a.prefix_max);
    LLM_REQUIRE(a.max_prefix >= 0 && a.max_prefix <= a.prefix_max, "%s: prefix of %d positions in a cache of %d", name, a.max_prefix, a.prefix_max);
    LLM_REQUIRE(a.max_tail >= 0 && a.max_tail < a.max_pos, "%s: %d rows behind the prefix in caches of %d", name, a.max_tail, a.max_pos);
    LLM_REQUIRE(a.ldq % 8 == 0 && a.ldq >= (n_heads + 2 * a.n_kv_heads) * head_dim && a.ldo >= n_heads * head_dim, "%s: ldq=%d ldo=%d", name,
                a.ldq, a.ldo);
    LLM_REQUIRE(aligned16(a.qkv) && aligned16(a.table) && aligned16(workspace) && a.prefix_offset % 8 == 0 && a.cache_offset % 8 == 0,
                "%s: qkv, table, workspace and the cache offsets must be 16-byte aligned", name);
    return LLM_OK;
}

extern "C" {

size_t llm_attn_shared_workspace_bytes(int n_heads, int n_kv_heads, int head_dim, int batch) {
    if (n_heads < 1 || n_kv_heads < 1 || head_dim < 1 || batch < 1) return 16;
    // at most as_target spans of the prefix, with batch rows per head, and as many of the tails
    const size_t target = (size_t)as_target(n_kv_heads, batch);
    return sizeof(float) * n_heads * target * (batch + 1) * (head_dim + 2);
}

int llm_attn_decode_rope_shared(const uint16_t *qkv, int ldq, const uint16_t *k_prefix, const uint16_t *v_prefix, int prefix_len,
                                int prefix_max_pos, uint16_t *const *k_caches, uint16_t *const *v_caches, const int *positions,
                                int row0, int batch, uint16_t *out, int ldo, const float *table, int n_heads, int n_kv_heads,
                                int head_dim, int max_pos, void *workspace, llm_stream_t stream) {
    const char *name = "llm_attn_decode_rope_shared";
    LLM_REQUIRE(k_caches && v_caches && positions && (prefix_len == 0 || (k_prefix && v_prefix)), "%s: null pointer", name);
    SharedArgs a = {};
    a.qkv = (const half_t *)qkv;
    a.ldq = ldq;
    a.out = (half_t *)out;
    a.ldo = ldo;
    a.table = table;
    a.batch = batch;
    a.n_kv_heads = n_kv_heads;
    a.max_pos = max_pos;
    a.prefix_max = prefix_max_pos;
    a.max_prefix = prefix_len;
    int rc = shared_check(name, a, n_heads, head_dim, workspace);
    if (rc != LLM_OK) return rc;
    LLM_REQUIRE(aligned16(k_prefix) && aligned16(v_prefix), "%s: the prefix caches must be 16-byte aligned", name);
    LLM_REQUIRE(row0 >= 0 && row0 <= prefix_len, "%s: row 0 of the caches holds position %d, behind the prefix of %d", name, row0, prefix_len);
    a.host.k_prefix = k_prefix;
    a.host.v_prefix = v_prefix;
    a.host.prefix_len = prefix_len;
    a.host.row0 = row0;
    for (int z = 0; z < batch; ++z) {
        LLM_REQUIRE(k_caches[z] && v_caches[z] && aligned16(k_caches[z]) && aligned16(v_caches[z]), "%s: cache %d", name, z);
        LLM_REQUIRE(positions[z] >= prefix_len && (long long)positions[z] - row0 < max_pos, "%s: position %d (the prefix has %d, the caches hold %d..%lld)",
                    name, positions[z], prefix_len, row0, (long long)row0 + max_pos - 1);
        for (int y = 0; y < z; ++y)
            LLM_REQUIRE(k_caches[y] != k_caches[z] && v_caches[y] != v_caches[z], "%s: sequences %d and %d share a cache", name, y, z);
        a.host.seq.k_cache[z] = k_caches[z];
        a.host.seq.v_cache[z] = v_caches[z];
        a.host.seq.pos[z] = positions[z];
        const int tail = positions[z] - prefix_len;
        a.max_tail = tail > a.max_tail ? tail : a.max_tail;
    }
    return dispatch_shared(name, a, n_heads, head_dim, workspace, (hipStream_t)stream);
}

int llm_attn_decode_rope_shared_dev(const uint16_t *qkv, int ldq, const llm_shared_desc *desc_dev, size_t prefix_offset,
                                    size_t cache_offset, int max_prefix, int prefix_max_pos, int max_tail, int batch, uint16_t *out,
                                    int ldo, const float *table, int n_heads, int n_kv_heads, int head_dim, int max_pos,
                                    void *workspace, llm_stream_t stream) {
    const char *name = "llm_attn_decode_rope_shared_dev";
    LLM_REQUIRE(desc_dev, "%s: null pointer", name);
    SharedArgs a = {};
    a.qkv = (const half_t *)qkv;
    a.ldq = ldq;
    a.out = (half_t *)out;
    a.ldo = ldo;
    a.table = table;
    a.batch = batch;
    a.n_kv_heads = n_kv_heads;
    a.max_pos = max_pos;
    a.prefix_max = prefix_max_pos;
    a.max_prefix = max_prefix;
    a.max_tail = max_tail;
    a.desc = desc_dev;
    a.prefix_offset = prefix_offset;
    a.cache_offset = cache_offset;
    int rc = shared_check(name, a, n_heads, head_dim, workspace);
    if (rc != LLM_OK) return rc;
    return dispatch_shared(name, a, n_heads, head_dim, workspace, (hipStream_t)stream);
}

} // extern "C"
