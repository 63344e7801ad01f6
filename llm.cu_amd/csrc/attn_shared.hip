// Decode attention of a batch whose sequences share their first positions: one new token per sequence, RoPE and the
// cache append of that token folded in.
//
//   score(z, h, j) = q'(z, h) . K(j) / sqrt(hd),   out(z, h) = sum_j softmax_j(score) V(j)
//
// Positions 0..prefix_len-1 come from one prefix cache, positions prefix_len..p_z-1 from the sequence's own cache (row r
// holds position row0 + r), position p_z is the new token, whose rotated key and value are appended to the own cache.
#include <cfloat>
#include <cmath>
#include <type_traits>

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
#define AS_RING 2     // stages, of 32 KB at most
#define AS_PER_CU 2   // workgroups that a compute unit holds
#define AS_LDS_PTR(p) ((__attribute__((address_space(3))) void *)(p))
#define AS_GLOBAL_PTR(p) ((const __attribute__((address_space(1))) void *)(p))

template <int HD, int QT> struct AsShape {
    static constexpr int SK = HD >= 128 ? 64 : 128;      // keys per stage
    static constexpr int KG = SK / 32 < AS_WAVES / QT ? SK / 32 : AS_WAVES / QT;
    static constexpr int DH = AS_WAVES / (QT * KG);
    static constexpr int NCH = SK / 32 / KG;             // chunks of a stage per wavefront
    static constexpr int TILE = SK * HD;                 // halves of a K or V^T tile
    static constexpr int NS = AS_RING;                   // stages of the ring
    static constexpr int DT = HD / 32 / DH;              // 32-dim tiles of the output per wavefront
    static_assert(QT * KG * DH == AS_WAVES && NCH >= 1 && DT >= 1, "roles of the wavefronts");
};
template <int HD> constexpr int as_lds_halves() { return AsShape<HD, 1>::NS * 2 * AsShape<HD, 1>::TILE; }

// Who does what.  The rows of a KV head -- the prefix, then each sequence's own rows -- form one line of units of 64 keys, with
// AS_START empty units in front of every tail (what starting on it costs), and the workgroups of the head take equal shares of the line,
// whatever the lengths are.  A workgroup leaves one part for each piece of the line that its share touches: part i of the
// prefix comes from workgroup i, and workgroup i's part of tail z goes to place i + z (both only grow along the line).
#define AS_UNIT 64
#define AS_START 3
struct AsPlan {
    int wgs, min_share; // workgroups per KV head; units a share has at least
    float *acc, *ml;    // [kvh][wgs][batch * G] of the prefix, then [kvh][wgs + batch][G] of the tails: rows of HD (acc), 2 (ml)
};
struct AsLine {
    int prefix_units, share, prefix, own_first, lead; // own_first: own row of the first position behind the prefix; lead: rows in
                                                      // front of it in the aligned eight that it lies in
    int tail, first, units;                           // lane z: own rows of sequence z, its first unit, its units
};
// Every lane of a wavefront calls it; lane z looks at sequence z.
template <bool DEV> __device__ __forceinline__ AsLine as_line(const SharedArgs &a, int batch, int wgs, int min_share) {
    const int lane = threadIdx.x % 64;
    const SharedSeq s = shared_seq<DEV>(a, lane < batch ? lane : 0);
    AsLine ln;
    ln.prefix = __builtin_amdgcn_readfirstlane(s.prefix);
    ln.own_first = __builtin_amdgcn_readfirstlane(s.first);
    ln.lead = ln.own_first & 7;
    ln.prefix_units = (ln.prefix + AS_UNIT - 1) / AS_UNIT;
    ln.tail = lane < batch ? s.tail : 0;
    ln.units = ln.tail > 0 ? (ln.lead + ln.tail + AS_UNIT - 1) / AS_UNIT : 0;
    int end = ln.units > 0 ? ln.units + AS_START : 0; // inclusive sums over the sequences
#pragma unroll
    for (int o = 1; o < LLM_MAX_BATCH; o <<= 1) {
        const int q = __shfl_up(end, o);
        if (lane >= o) end += q;
    }
    ln.first = ln.prefix_units + end - ln.units;
    const int total = ln.prefix_units + __builtin_amdgcn_readlane(end, LLM_MAX_BATCH - 1);
    ln.share = (total + wgs - 1) / wgs;
    if (ln.share < min_share) ln.share = min_share;
    return ln;
}

// Rows of one part: tiles from `begin` (a multiple of eight) on, of which rows lo .. hi - 1 count.
struct AsRange {
    int begin, lo, hi;
};

// q_row(r): query row r of the tiles, not rotated (any r below 32 QT); q_seq(r): its row of the (cos, sin) table's rows that
// are staged, cs_row(i), i < LLM_MAX_BATCH.
template <int HD, int QT, class QRow, class QSeq, class CsRow>
__device__ __forceinline__ void as_span(half_t *smem, const half_t *kbase, const half_t *vbase, const int max_pos, const AsRange r,
                                        const int rows, QRow q_row, QSeq q_seq, CsRow cs_row, float *acc, float *ml) {
    using S = AsShape<HD, QT>;
    constexpr int SK = S::SK, KG = S::KG, DH = S::DH, NS = S::NS, DT = S::DT, TILE = S::TILE;
    constexpr int NC = HD / 8, NCV = SK / 8, NCC = HD / 4;       // 16-byte chunks per K row / V^T row of a tile / row of the table
    constexpr int LPW = TILE * 2 / 1024 / AS_WAVES;              // loads per wavefront, stage and tile (1 KB each)
    constexpr int Q_HALVES = 32 * QT * HD, CS_HALVES = LLM_MAX_BATCH * HD * 2;
    constexpr int NQ = Q_HALVES + CS_HALVES <= 2 * TILE ? 1 : 2; // last slots of the ring that hold queries and table rows first
    static_assert(AS_WAVES * (64 / NC) % 16 == 0 && AS_WAVES * (64 / NCV) % 16 == 0, "the swizzle is the same for all loads of a lane");
    static_assert(Q_HALVES + CS_HALVES <= NQ * 2 * TILE && NQ <= NS, "room for the queries");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const int qt = wave % QT, kg = wave / QT % KG, dh = wave / (QT * KG);
    const int n = lane % 32, hb = lane / 32;
    const int stages = (r.hi - r.begin + SK - 1) / SK;

    // ---- loads: instruction i of a wavefront covers rows 4 i + wave, in units of the rows that 1 KB holds ----
    const __amdgpu_buffer_rsrc_t rs_k = __builtin_amdgcn_make_buffer_rsrc((void *)kbase, 0, max_pos * HD * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t rs_v = __builtin_amdgcn_make_buffer_rsrc((void *)vbase, 0, HD * max_pos * 2, 0x00020000);
    auto swz = [](int row, int chunks) { return chunks >= 16 ? row & 15 : row / (16 / chunks) & (chunks - 1); }; // of 16-byte chunks over the banks
    const int krow = wave * (64 / NC) + lane / NC, vrow = wave * (64 / NCV) + lane / NCV;
    const int kchunk = lane % NC ^ swz(krow, NC), vchunk = lane % NCV ^ swz(vrow, NCV);
    const uint32_t koff = (uint32_t)krow * (HD * 2) + (uint32_t)kchunk * 16;
    const uint32_t voff = (uint32_t)vrow * (uint32_t)max_pos * 2u + (uint32_t)vchunk * 16;
    auto issue = [&](int slot, int st) __attribute__((always_inline)) { // stage st into slot % NS of the ring
        half_t *buf = smem + slot % NS * 2 * TILE;
        const int key = r.begin + st * SK;
        if (key + SK <= r.hi) {
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
        // the tile reaches past the last row that counts: what lies behind is read from that one (and masked later)
        const int vkey = key + 8 * vchunk < r.hi ? key + 8 * vchunk : (r.hi - 1) & ~7;
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
            const int row = key + i * AS_WAVES * (64 / NC) + krow;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_k, AS_LDS_PTR(buf + (i * AS_WAVES + wave) * 512), 16,
                                                     (uint32_t)(row < r.hi ? row : r.hi - 1) * (HD * 2) + (uint32_t)kchunk * 16, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < LPW; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_v, AS_LDS_PTR(buf + TILE + (i * AS_WAVES + wave) * 512), 16,
                                                     ((uint32_t)(i * AS_WAVES * (64 / NCV) + vrow) * (uint32_t)max_pos + (uint32_t)vkey) * 2u, 0, 0, 0);
    };

    // ---- queries and the (cos, sin) rows of their positions: through the last slots of the ring, like the tiles and in front
    // of them, so that no load into registers is waited for behind the tiles' (loads complete in order: that would be a wait
    // for the whole ring) ----
    half_t *q_l = smem + (NS - NQ) * 2 * TILE, *cs_l = q_l + Q_HALVES;
    for (int i = wave; i < Q_HALVES / 512; i += AS_WAVES) { // 1 KB: 64 / NC rows, swizzled like a K tile
        const int row = i * (64 / NC) + lane / NC;
        __builtin_amdgcn_global_load_lds(AS_GLOBAL_PTR(q_row(row) + (lane % NC ^ swz(row, NC)) * 8), AS_LDS_PTR(q_l + i * 512), 16, 0, 0);
    }
    for (int i = wave; i < CS_HALVES / 512; i += AS_WAVES) {
        const int row = i * (64 / NCC) + lane / NCC;
        __builtin_amdgcn_global_load_lds(AS_GLOBAL_PTR(cs_row(row) + (lane % NCC ^ (row & (NCC - 1) & 15)) * 4), AS_LDS_PTR(cs_l + i * 512), 16, 0, 0);
    }
    // always NS stages (a short piece's last one more than once): the number of loads in flight is known everywhere
    const int issued = stages > NS ? stages : NS;
#pragma unroll
    for (int st = 0; st < NS - NQ; ++st) issue(st, st < stages ? st : stages - 1);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - NQ) * 2 * LPW) : "memory");
    half8_t qf[HD / 16]; // lane (n, hb) holds dims 16 ks + 8 hb .. + 7 of row 32 qt + n
    {
        const int row = 32 * qt + n, z = q_seq(row);
        float4_t cs[HD / 16][2];
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
            qf[ks] = load8(q_l + row * HD + ((2 * ks + hb) ^ swz(row, NC)) * 8);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                cs[ks][i] = *reinterpret_cast<const float4_t *>(cs_l + z * HD * 2 + ((4 * ks + 2 * hb + i) ^ (z & (NCC - 1) & 15)) * 8);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); // every wavefront has its queries: the slots are free
#pragma unroll
        for (int st = NS - NQ; st < NS; ++st) issue(st, st < stages ? st : stages - 1);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) { // rotated while the tiles travel
            float c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = cs[ks][i / 4][i % 4];
            qf[ks] = rope_rotate8(qf[ks], c);
        }
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
        half_t *ks_ = smem + st % NS * 2 * TILE, *vs_ = ks_ + TILE;
        const int key_st = r.begin + st * SK;
        const bool edge = key_st < r.lo || key_st + SK > r.hi;
        if (edge) { // values outside the piece's rows may be anything, NaN included: zero in the tile
            for (int i = tid; i < HD * NCV; i += AS_THREADS) {
                const int dim = i / NCV, c = i % NCV, k0 = key_st + 8 * c;
                if (k0 >= r.lo && k0 + 8 <= r.hi) continue;
                half_t *at = vs_ + dim * SK + (c ^ swz(dim, NCV)) * 8;
                half8_t v = load8(at);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = k0 + e >= r.lo && k0 + e < r.hi ? v[e] : (half_t)0.f;
                store8(at, v);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
#pragma unroll
        for (int j = 0; j < S::NCH; ++j) {
            const int kc = 32 * (kg + KG * j), key0 = key_st + kc;   // the chunk in the stage; its first key
            if (key0 >= r.hi || key0 + 32 <= r.lo) continue;        // no key of the piece (the same for every lane)
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
                    const half8_t vf = load8(vs_ + dim * SK + ((kc / 8 + 2 * u + hb) ^ swz(dim, NCV)) * 8);
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

// Grid: wgs x KV heads, the KV head fastest: consecutive workgroups go round the XCDs, so that a head's queries and tables stay
// in one XCD's L2.  The arguments in front of `a` are in registers when the kernel starts.
template <int HD, int G, int QT, bool DEV>
__global__ __launch_bounds__(AS_THREADS, AS_WAVES * AS_PER_CU / 4) void attn_shared_part_kernel(float *acc, float *ml, const half_t *qkv, const float *table, int n_kv_heads,
                                                                      int batch, int wgs, int min_share, int ldq, int prefix_max,
                                                                      const SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) half_t smem[];
    const int kvh = blockIdx.x % n_kv_heads, wg = blockIdx.x / n_kv_heads;
    const int rows = batch * G;
    const SharedSeq s0 = shared_seq<DEV>(a, 0); // asked for next to the positions that the line needs
    const AsLine ln = as_line<DEV>(a, batch, wgs, min_share);
    const int from = wg * ln.share, to = from + ln.share; // this workgroup's units
    if (from < ln.prefix_units) {
        const int end = to * AS_UNIT < ln.prefix ? to * AS_UNIT : ln.prefix;
        const size_t at = ((size_t)kvh * wgs + wg) * rows;
        auto q_row = [&](int row) {
            row = row < rows ? row : rows - 1;
            return qkv + (size_t)(row / G) * ldq + (size_t)(kvh * G + row % G) * HD;
        };
        auto q_seq = [&](int row) { return row < rows ? row / G : batch - 1; };
        auto cs_row = [&](int z) { return table + (size_t)(ln.prefix + __shfl(ln.tail, z)) * HD; };
        as_span<HD, QT>(smem, s0.kp + (size_t)kvh * prefix_max * HD, s0.vp + (size_t)kvh * HD * prefix_max, prefix_max,
                        AsRange{from * AS_UNIT, from * AS_UNIT, end}, rows, q_row, q_seq, cs_row, acc + at * HD, ml + at * 2);
    }
    unsigned long long mine = __builtin_amdgcn_ballot_w64(ln.units > 0 && ln.first < to && ln.first + ln.units > from); // tails
    for (; mine; mine &= mine - 1) {
        const int z = __builtin_ctzll(mine);
        const int first = __builtin_amdgcn_readlane(ln.first, z), u = __builtin_amdgcn_readlane(ln.units, z), tail = __builtin_amdgcn_readlane(ln.tail, z);
        const int u0 = from > first ? from - first : 0, u1 = to - first < u ? to - first : u;
        const int base = ln.own_first - ln.lead, b = base + u0 * AS_UNIT, e = base + u1 * AS_UNIT, end = ln.own_first + tail;
        const size_t at = (size_t)n_kv_heads * wgs * rows + ((size_t)kvh * (wgs + batch) + wg + z) * G;
        const SharedSeq s = shared_seq<DEV>(a, z);
        auto q_row = [&](int row) { return qkv + (size_t)z * ldq + (size_t)(kvh * G + (row < G ? row : G - 1)) * HD; };
        auto q_seq = [&](int) { return 0; };
        auto cs_row = [&](int) { return table + (size_t)(ln.prefix + tail) * HD; };
        __syncthreads(); // the LDS of the piece before
        as_span<HD, 1>(smem, s.kc + (size_t)kvh * a.max_pos * HD, s.vc + (size_t)kvh * HD * a.max_pos, a.max_pos,
                       AsRange{b, b > ln.own_first ? b : ln.own_first, e < end ? e : end}, G, q_row, q_seq, cs_row, acc + at * HD, ml + at * 2);
    }
}

// One workgroup per query head and sequence: the parts' weights (first wavefront) and the new token's score (second one) while
// the parts' rows travel, then the weighted sum.  The first head of a group appends the new key and value.
#define AS_MERGE_THREADS 256
#define AS_MERGE_AHEAD 8
template <int HD, int G, bool DEV>
__global__ __launch_bounds__(AS_MERGE_THREADS) void attn_shared_merge_kernel(const float *acc, const float *ml, const half_t *qkv, const float *table,
                                                                             int n_kv_heads, int batch, int wgs, int min_share, int ldq, int max_pos,
                                                                             const SharedArgs a) {
    constexpr int LPR = HD / 4, GROUPS = AS_MERGE_THREADS / LPR; // lanes per row of HD floats, rows side by side
    extern __shared__ float weight[]; // one per part
    __shared__ float m_parts, l_parts, m_new;
    __shared__ float4_t part[GROUPS][LPR];
    const int h = blockIdx.x, z = blockIdx.y, kvh = h / G, g = h % G, tid = threadIdx.x, lane = tid % 64;
    const int rows = batch * G, Hq = n_kv_heads * G;
    const SharedSeq s = shared_seq<DEV>(a, z);
    const int pos = s.prefix + s.tail, row = s.first + s.tail;
    const AsLine ln = as_line<DEV>(a, batch, wgs, min_share);
    const int first = __builtin_amdgcn_readlane(ln.first, z), u = __builtin_amdgcn_readlane(ln.units, z);
    const int np = (ln.prefix_units + ln.share - 1) / ln.share;
    const int w0 = first / ln.share, nt = u > 0 ? (first + u - 1) / ln.share - w0 + 1 : 0, ns = np + nt;
    const size_t pre = (size_t)kvh * wgs * rows + (size_t)z * G + g;
    const size_t own = (size_t)n_kv_heads * wgs * rows + ((size_t)kvh * (wgs + batch) + w0 + z) * G + g;
    auto slot = [&](int i) { return i < np ? pre + (size_t)i * rows : own + (size_t)(i - np) * G; };
    const half_t *line = qkv + (size_t)z * ldq;
    const half_t *vn = line + (size_t)(Hq + n_kv_heads + kvh) * HD;
    const int d4 = tid % LPR, grp = tid / LPR;
    float4_t v[AS_MERGE_AHEAD];
#pragma unroll
    for (int j = 0; j < AS_MERGE_AHEAD; ++j) {
        v[j] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (grp + GROUPS * j < ns) v[j] = *reinterpret_cast<const float4_t *>(acc + slot(grp + GROUPS * j) * HD + 4 * d4);
    }
    if (tid < 64) {
        float M = -FLT_MAX, l = 0.f;
        for (int i = lane; i < ns; i += 64) {
            const float2_t p = *reinterpret_cast<const float2_t *>(ml + 2 * slot(i));
            // relative to this lane's largest so far
            const float m = fmaxf(M, p[0]);
            l = l * __builtin_amdgcn_exp2f(M - m) + p[1] * __builtin_amdgcn_exp2f(p[0] - m);
            M = m;
            weight[i] = p[0];
        }
        const float all = wave_max(M);
        l = wave_sum(l * __builtin_amdgcn_exp2f(M - all));
        for (int i = lane; i < ns; i += 64) weight[i] = __builtin_amdgcn_exp2f(weight[i] - all);
        if (lane == 0) {
            m_parts = all;
            l_parts = l;
        }
    } else if (tid < 128) {
        float dot = 0.f;
        if (lane < HD / 8) { // eight dims per lane
            const float *cs = table + (size_t)pos * HD + lane * 8;
            const half8_t q = rope_rotate8(load8(line + (size_t)h * HD + lane * 8), cs);
            const half8_t k = rope_rotate8(load8(line + (size_t)(Hq + kvh) * HD + lane * 8), cs);
            dot = dot8(q, k, 0.f);
            if (g == 0) {
                store8(s.kc + ((size_t)kvh * max_pos + row) * HD + lane * 8, k);
                const half8_t vv = load8(vn + lane * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) s.vc[((size_t)kvh * HD + lane * 8 + e) * max_pos + row] = vv[e];
            }
        }
        dot = wave_sum(dot) * (1.44269504088896341f / sqrtf((float)HD));
        if (lane == 0) m_new = dot;
    }
    __syncthreads();
    float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < AS_MERGE_AHEAD; ++j) {
        if (grp + GROUPS * j < ns) {
            const float w = weight[grp + GROUPS * j];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += w * v[j][e];
        }
    }
    for (int i = grp + GROUPS * AS_MERGE_AHEAD; i < ns; i += GROUPS) {
        const float4_t x = *reinterpret_cast<const float4_t *>(acc + slot(i) * HD + 4 * d4);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += weight[i] * x[e];
    }
    part[grp][d4] = o;
    __syncthreads();
    if (tid < LPR) {
        const float M = fmaxf(m_parts, m_new), f = __builtin_amdgcn_exp2f(m_parts - M), w = __builtin_amdgcn_exp2f(m_new - M);
        const float inv = 1.0f / (f * l_parts + w);
        const half4_t x = *reinterpret_cast<const half4_t *>(vn + 4 * d4);
        half_t *out = a.out + (size_t)z * a.ldo + (size_t)h * HD + 4 * d4;
        o = part[0][d4];
#pragma unroll
        for (int i = 1; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += part[i][d4][e];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = (half_t)((f * o[e] + w * (float)x[e]) * inv);
    }
}

// Workgroups per KV head: one on each of the 256 compute units.
static int as_wgs(int n_kv_heads) { return n_kv_heads < 256 * AS_PER_CU ? 256 * AS_PER_CU / n_kv_heads : 1; }

template <int HD, int G, int QT, bool DEV> static int launch_shared(const SharedArgs &a, const AsPlan &pl, hipStream_t s) {
    const size_t smem = sizeof(half_t) * as_lds_halves<HD>();
    auto kern = attn_shared_part_kernel<HD, G, QT, DEV>;
    static std::atomic<uint64_t> attr_done{0};
    if (smem > 48 * 1024) {
        int rc = llm_ensure_max_smem((const void *)kern, smem, attr_done);
        if (rc != LLM_OK) return rc;
    }
    // no more workgroups than the longest lengths of the launch give shares to
    const long long units = (a.max_prefix + AS_UNIT - 1) / AS_UNIT +
                            (a.max_tail > 0 ? (long long)a.batch * ((a.max_tail + 7 + AS_UNIT - 1) / AS_UNIT + AS_START) : 0);
    long long used = (units + pl.min_share - 1) / pl.min_share;
    if (used > pl.wgs) used = pl.wgs;
    if (used > 0) {
        kern<<<dim3((unsigned)used * a.n_kv_heads), dim3(AS_THREADS), smem, s>>>(pl.acc, pl.ml, a.qkv, a.table, a.n_kv_heads, a.batch, pl.wgs,
                                                                                   pl.min_share, a.ldq, a.prefix_max, a);
        LLM_LAUNCH_CHECK("attn_shared_part_kernel");
    }
    attn_shared_merge_kernel<HD, G, DEV><<<dim3(a.n_kv_heads * G, a.batch), dim3(AS_MERGE_THREADS), sizeof(float) * 2 * (pl.wgs + 1), s>>>(
        pl.acc, pl.ml, a.qkv, a.table, a.n_kv_heads, a.batch, pl.wgs, pl.min_share, a.ldq, a.max_pos, a);
    LLM_LAUNCH_CHECK("attn_shared_merge_kernel");
    return LLM_OK;
}

template <int HD, int G> static int launch_shared(const SharedArgs &a, void *ws, hipStream_t s) {
    const int rows = a.batch * G;
    AsPlan pl = {};
    pl.wgs = as_wgs(a.n_kv_heads);
    pl.min_share = 2;
    pl.acc = (float *)ws;
    pl.ml = pl.acc + (size_t)a.n_kv_heads * ((size_t)pl.wgs * rows + (size_t)(pl.wgs + a.batch) * G) * HD;
    constexpr int MAXR = G * LLM_MAX_BATCH;
    // as many query tiles as the batch fills
    if (rows <= 32 || MAXR <= 32) return a.desc ? launch_shared<HD, G, 1, true>(a, pl, s) : launch_shared<HD, G, 1, false>(a, pl, s);
    if (rows <= 64 || MAXR <= 64) return a.desc ? launch_shared<HD, G, MAXR >= 64 ? 2 : 1, true>(a, pl, s) : launch_shared<HD, G, MAXR >= 64 ? 2 : 1, false>(a, pl, s);
    return a.desc ? launch_shared<HD, G, MAXR >= 128 ? 4 : 1, true>(a, pl, s) : launch_shared<HD, G, MAXR >= 128 ? 4 : 1, false>(a, pl, s);
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
    const size_t wgs = (size_t)as_wgs(n_kv_heads);
    return sizeof(float) * n_heads * (wgs * batch + wgs + batch) * (head_dim + 2);
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
