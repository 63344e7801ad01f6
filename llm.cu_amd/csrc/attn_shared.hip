// Decode attention of a batch whose sequences share their first positions: one new token per sequence, RoPE and the
// cache append of that token folded in.
//
//   score(z, h, j) = q'(z, h) . K(j) / sqrt(hd),   out(z, h) = sum_j softmax_j(score) V(j)
//
// Positions 0..prefix_len-1 come from one prefix cache, positions prefix_len..p_z-1 from the sequence's own cache (row r
// holds position row0 + r), position p_z is the new token, whose rotated key and value are appended to the own cache.
//
// What bounds it: the bytes of the caches.  Per KV head and prefix position 2 hd halves are read for 4 hd batch G operations (6 hd
// with the second half of the weights), 64 (96) operations a byte at 16 sequences with four query heads each, where this chip's
// matrix pipe does about 240 per byte of memory traffic: read once, the prefix costs its bytes.  One sequence at a time would read it `batch` times.
// Measured, 32 / 8 heads of 128, 16 sequences, one call (two launches): 8192 + 256 positions each 18.5 us (43 MB, 8.5 us at the
// 5.07 TB/s of a large copy), 32768 + 1024 46.6 us (171 MB, 33.8 us); llm_attn_decode_rope_batch on caches of their own 108 us
// at 16 x 8192.  In its steady state the first launch reads 6.3 TB/s; what is left hardly depends on the lengths: 4 to 5 us until
// its first tiles are there (half of the ring holds queries and table rows first), 1.5 us at its end, 5 to 6 us for the second launch
// and the parts in front of it (16.8 MB written and read when 512 workgroups leave some for 16 sequences).
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "ranges.hpp"

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
    int prefix = d.prefix_len, row0 = d.row0, tail = (int)((uint32_t)d.seq.pos[z] - (uint32_t)d.prefix_len);
    if (DEV) {
        prefix = prefix < 0 ? 0 : prefix > a.max_prefix ? a.max_prefix : prefix;
        row0 = row0 < 0 ? 0 : row0 > prefix ? prefix : row0;
        if (prefix - row0 > a.max_pos - 1) prefix = row0 + a.max_pos - 1; // positions stay below row0 + max_pos, as the table does
        const int most = a.max_tail < a.max_pos - 1 - (prefix - row0) ? a.max_tail : a.max_pos - 1 - (prefix - row0);
        tail = tail < 0 ? 0 : tail > most ? most : tail;
    }
    s.prefix = prefix;
    s.first = prefix - row0;
    s.tail = tail;
    return s;
}

// ---------------------------------------------------------------------------------------------------------------
// Parts.  A workgroup takes one KV head and runs of its cache rows: of the prefix, for the queries of all sequences (batch * G
// rows in QT tiles of 32), or of one sequence's own rows, for its G queries.  It leaves, per query row, the reference maximum,
// the sum and the unnormalised P.V; attn_shared_merge_kernel joins the parts and adds the new token.
//
// The products are the transposed ones of the prompt pass: S^T = K . Q^T and O^T += V^T . P^T on v_mfma_f32_32x32x16_f16, so that
// a lane holds one query's column and the accumulators of the first product are the operand of the second: with the K rows of a
// 32-key chunk read in the order pi(m) (bits 2 and 3 of m swapped), accumulator e of lane (n, hb) is key 16 (e / 8) + 8 hb + e % 8.
//
// K and V^T tiles of SK keys travel straight into a ring of LDS stages (buffer_load ... lds); a lane fetches the 16-byte chunk
// that the bank swizzle assigns to its slot.  The four wavefronts of a workgroup are QT query tiles x KG groups of keys x DH
// parts of the output dims (DH = 2: both compute the scores, each half of the output).
//
// Two workgroups of four wavefronts per compute unit, each with a ring of two 32 KB stages, so that one works or begins while the
// other waits: 45.3 / 21.0 us at 16 x (32768 + 1024) / (8192 + 256) against 47.8 / 22.8 us with one workgroup of eight
// wavefronts and four stages (weights in one operand, shares of two units).
// ---------------------------------------------------------------------------------------------------------------
#define AS_WAVES 4    // wavefronts of a workgroup
#define AS_THREADS (64 * AS_WAVES)
#define AS_RING 2     // stages
#define AS_PER_CU 2   // workgroups that a compute unit holds
#define AS_LDS_PTR(p) ((__attribute__((address_space(3))) void *)(p))
#define AS_GLOBAL_PTR(p) ((const __attribute__((address_space(1))) void *)(p))

template <int HD, int QT, int W> struct AsShape { // W wavefronts
    static constexpr int SK = (HD >= 128 ? 16 : 32) * W; // keys per stage
    static constexpr int KG = SK / 32 < W / QT ? SK / 32 : W / QT;
    static constexpr int DH = W / (QT * KG);
    static constexpr int NCH = SK / 32 / KG;             // chunks of a stage per wavefront
    static constexpr int TILE = SK * HD;                 // halves of a K or V^T tile
    static constexpr int NS = AS_RING;                   // stages of the ring
    static constexpr int DT = HD / 32 / DH;              // 32-dim tiles of the output per wavefront
    static_assert(QT * KG * DH == W && NCH >= 1 && DT >= 1, "roles of the wavefronts");
};
// LDS: the ring, and in its place at the end what the wavefronts hold: four accumulators of every lane form a block, lane (n, hb)
// at n + 40 hb of its 73 places of 16 bytes, so that neither a block nor a query row's dims in order meet on the banks.
#define AS_BLOCK 73
#define AS_HALF 40
template <int HD, int QT, int W> constexpr int as_held() { return 4 * AsShape<HD, QT, W>::DT * AS_BLOCK * 4 + 128; } // floats of a wavefront
template <int HD, int QT, int W> constexpr int as_lds_bytes() {
    constexpr int ring = AsShape<HD, QT, W>::NS * 4 * AsShape<HD, QT, W>::TILE, held = W * as_held<HD, QT, W>() * 4;
    return ring > held ? ring : held;
}

// Who does what.  The rows of a KV head -- the prefix, then each sequence's own rows -- form one line of units of 64 keys, with
// `start` empty units in front of every tail (what starting on it costs), and the workgroups of the head take equal shares of the
// line, whatever the lengths are.  A workgroup leaves one part for each piece of the line that its share touches: part i of the
// prefix comes from workgroup i, and workgroup i's part of tail z goes to place i + z (both only grow along the line).
//
// Whole tiles: in units of 8, 16 and 32 keys, whose shares are nearer to equal but end inside a tile, 16 x (32768 + 1024) took
// 47.6, 47.4 and 46.5 us against 45.3, 16 x (8192 + 256) 23.9, 23.6 and 23.3 us against 21.0 (weights in one operand, shares of two
// units).
//
// A share's size.  A unit costs its workgroup some 1 us as long as memory is not full, a part costs every row of the merge: the
// best size grows with the square root of the line, and with that of the KV heads, whose parts the merge reads side by side.
// Measured with 8 heads of 128, shares of 2, 3, 4, 5, 6, 8 and 10 units: 2 x (2048 + 16) 10.7 10.8 11.5 12.4 13.3 15.2 17.0 us,
// 2 x (4096 + 64) 12.8 11.5 11.9 12.7 13.6 15.4 17.3, 2 x (8192 + 64) 15.0 (3 units at least) 15.0 13.6 13.4 13.8 15.6 17.4,
// 4 x (16384 + 64) 19.8 (5 at least) .. 20.3 17.6 18.2.  One KV head: 4 x (32768 + 100) 22.7 us with 2 units, 16.2 with 4, 15.3 with 5,
// 19.5 with 11.  From 16384 positions on all workgroups are wanted, at the smaller heads (half the bytes and less per unit) always:
// 8 heads of 64, 4 x (32768 + 100) 18.8 us with 8 units, 20.1 with 11.
//
// Empty units: 6, 3 where memory is full and a unit takes three times as long: with 3 and 6, 16 x (8192 + 64) 19.5 and 17.7 us,
// 8 x (8192 + 128) 16.5 and 15.0, 16 x (32768 + 1024) 46.6 and 47.7, 8 x (2048 + 64), in shares of two, 11.6 and 12.5.
#define AS_UNIT 64
struct AsPlan {
    int wgs;            // workgroups per KV head
    uint32_t inv;       // 2^32 / wgs, rounded up
    float *acc, *ml;    // [kvh][wgs][batch * G] of the prefix, then [kvh][wgs + batch][G] of the tails: rows of HD (acc), 2 (ml)
};
struct AsShare {
    int start, share; // empty units in front of a tail, units per workgroup
};
template <int HD> __host__ __device__ __forceinline__ AsShare as_share(int prefix_units, int tail_units, int tails, int n_kv_heads, int wgs,
                                                                             uint32_t inv) {
    int least = 2;
    const int size = prefix_units * (n_kv_heads < 8 ? n_kv_heads : 8);
    if (HD >= 128) {
#pragma unroll
        for (int m = 3; m <= 8; ++m) least += size >= 32 * m * m;
    }
    AsShare r;
    r.start = least >= 4 && prefix_units + tail_units + 3 * tails <= 6 * wgs ? 6 : 3;
    const uint32_t total = (uint32_t)(prefix_units + tail_units + r.start * tails);
    r.share = wgs > 1 ? (int)((uint64_t)(total + wgs - 1) * inv >> 32) : (int)total; // total / wgs, rounded up
    if (r.share < least) r.share = least;
    return r;
}
struct AsLine {
    int prefix_units, share, prefix, own_first, lead; // own_first: own row of the first position behind the prefix; lead: rows in
                                                      // front of it in the aligned eight that it lies in
    int tail, first, units;                           // lane z: own rows of sequence z, its first unit, its units
};
// Every lane of a wavefront calls it; lane z looks at sequence z.
template <int HD, bool DEV> __device__ __forceinline__ AsLine as_line(const SharedArgs &a, int n_kv_heads, int batch, int wgs,
                                                                                 uint32_t inv) {
    const int lane = threadIdx.x % 64;
    const SharedSeq s = shared_seq<DEV>(a, lane < batch ? lane : 0);
    AsLine ln;
    ln.prefix = __builtin_amdgcn_readfirstlane(s.prefix);
    ln.own_first = __builtin_amdgcn_readfirstlane(s.first);
    ln.lead = ln.own_first & 7;
    ln.prefix_units = (ln.prefix + AS_UNIT - 1) / AS_UNIT;
    ln.tail = lane < batch ? s.tail : 0;
    ln.units = ln.tail > 0 ? (ln.lead + ln.tail + AS_UNIT - 1) / AS_UNIT : 0;
    // inclusive sums over the sequences, the first row of 16 lanes (row_shr by 1, 2, 4, 8; zeros come in): a chain in front of every
    // load, 0.1 to 0.3 us of both launches shorter than by shuffles
    int end = ln.units;
    static_assert(LLM_MAX_BATCH == 16, "one row of lanes");
    end += __builtin_amdgcn_update_dpp(0, end, 0x111, 0xf, 0xf, true);
    end += __builtin_amdgcn_update_dpp(0, end, 0x112, 0xf, 0xf, true);
    end += __builtin_amdgcn_update_dpp(0, end, 0x114, 0xf, 0xf, true);
    end += __builtin_amdgcn_update_dpp(0, end, 0x118, 0xf, 0xf, true);
    const unsigned long long tails = __builtin_amdgcn_ballot_w64(ln.units > 0);
    const AsShare sh = as_share<HD>(ln.prefix_units, __builtin_amdgcn_readlane(end, LLM_MAX_BATCH - 1), __popcll(tails), n_kv_heads, wgs, inv);
    ln.share = sh.share;
    ln.first = ln.prefix_units + end - ln.units + sh.start * __popcll(tails & ((2ull << lane) - 1ull));
    return ln;
}

// A piece of the line: rows of one head's half-caches, in tiles from `begin` (a multiple of eight) on, of which lo .. hi - 1 count.
struct AsPiece {
    const half_t *k, *v;
    int max_pos, begin, lo, hi;
};

// References of exponentials are unscaled scores; as_c2 takes a difference of two to the base of exp2.
template <int HD> __device__ __forceinline__ float as_c2() { return 1.44269504088896341f / sqrtf((float)HD); }

// The tiles of NP pieces, one behind the other, for up to 32 QT query rows.
// q_row(r): query row r, not rotated (any r below 32 QT); q_seq(r): which of the staged rows cs_row(i), i < LLM_MAX_BATCH, of the
// (cos, sin) table is its position's.
// between(qf): called when the rotated query rows are there, lane (n, hb) holding dims 16 ks + 8 hb .. + 7 of row 32 qt + n;
// what it leaves in LDS outside the ring is visible behind as_tiles.
// Leaves every wavefront's output, maxima and sums in the LDS, behind a barrier, for as_result.
template <int HD, int QT, int W, int NP, class QRow, class QSeq, class CsRow, class Between>
__device__ __forceinline__ void as_tiles(half_t *smem, const AsPiece (&pc)[NP], QRow q_row, QSeq q_seq, CsRow cs_row, Between between) {
    using S = AsShape<HD, QT, W>;
    constexpr int SK = S::SK, KG = S::KG, DH = S::DH, NS = S::NS, DT = S::DT, TILE = S::TILE;
    constexpr int NC = HD / 8, NCV = SK / 8, NCC = HD / 4;       // 16-byte chunks per K row / V^T row of a tile / row of the table
    constexpr int LPW = TILE * 2 / 1024 / W;                     // loads per wavefront, stage and tile (1 KB each)
    constexpr int Q_HALVES = 32 * QT * HD, CS_HALVES = LLM_MAX_BATCH * HD * 2;
    constexpr int NQ = Q_HALVES + CS_HALVES <= 2 * TILE ? 1 : 2; // last slots of the ring that hold queries and table rows first
    static_assert(W * (64 / NC) % 16 == 0 && W * (64 / NCV) % 16 == 0, "the swizzle is the same for all loads of a lane");
    static_assert(Q_HALVES + CS_HALVES <= NQ * 2 * TILE && NQ <= NS, "room for the queries");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const int qt = wave % QT, kg = wave / QT % KG, dh = wave / (QT * KG);
    const int n = lane % 32, hb = lane / 32;
    const int stages_0 = (pc[0].hi - pc[0].begin + SK - 1) / SK; // of the first piece
    const int real = NP == 1 ? stages_0 : stages_0 + (pc[NP - 1].hi - pc[NP - 1].begin + SK - 1) / SK;
    const int stages = real > 0 ? real : 1;                      // no row at all: one tile that is masked throughout

    // ---- loads: instruction i of a wavefront covers rows W i + wave, in units of the rows that 1 KB holds ----
    auto swz = [](int row, int chunks) { return chunks >= 16 ? row & 15 : row / (16 / chunks) & (chunks - 1); }; // of 16-byte chunks over the banks
    const int krow = wave * (64 / NC) + lane / NC, vrow = wave * (64 / NCV) + lane / NCV;
    const int kchunk = lane % NC ^ swz(krow, NC), vchunk = lane % NCV ^ swz(vrow, NCV);
    const uint32_t koff = (uint32_t)krow * (HD * 2) + (uint32_t)kchunk * 16;
    auto first_key = [&](int st, const AsPiece &p) { return NP > 1 && &p != &pc[0] ? p.begin + (st - stages_0) * SK : p.begin + st * SK; };
    auto issue_of = [&](int slot, int st, const AsPiece &p) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rs_k = __builtin_amdgcn_make_buffer_rsrc((void *)p.k, 0, p.max_pos * HD * 2, 0x00020000);
        const __amdgpu_buffer_rsrc_t rs_v = __builtin_amdgcn_make_buffer_rsrc((void *)p.v, 0, HD * p.max_pos * 2, 0x00020000);
        half_t *buf = smem + slot % NS * 2 * TILE;
        const int key = first_key(st, p), hi = p.hi > 0 ? p.hi : 1;
        if (key + SK <= hi) {
            const uint32_t voff = (uint32_t)vrow * (uint32_t)p.max_pos * 2u + (uint32_t)vchunk * 16;
#pragma unroll
            for (int i = 0; i < LPW; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_k, AS_LDS_PTR(buf + (i * W + wave) * 512), 16, koff,
                                                         (uint32_t)key * (HD * 2) + (uint32_t)i * (W * 1024), 0, 0);
#pragma unroll
            for (int i = 0; i < LPW; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_v, AS_LDS_PTR(buf + TILE + (i * W + wave) * 512), 16, voff,
                                                         (uint32_t)key * 2 + (uint32_t)i * (W * (64 / NCV)) * (uint32_t)p.max_pos * 2u, 0, 0);
            return;
        }
        // the tile reaches past the last row that counts: what lies behind is read from that one (and masked later)
        const int vkey = key + 8 * vchunk < hi ? key + 8 * vchunk : (hi - 1) & ~7;
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
            const int row = key + i * W * (64 / NC) + krow;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_k, AS_LDS_PTR(buf + (i * W + wave) * 512), 16,
                                                     (uint32_t)(row < hi ? row : hi - 1) * (HD * 2) + (uint32_t)kchunk * 16, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < LPW; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_v, AS_LDS_PTR(buf + TILE + (i * W + wave) * 512), 16,
                                                     ((uint32_t)(i * W * (64 / NCV) + vrow) * (uint32_t)p.max_pos + (uint32_t)vkey) * 2u, 0, 0, 0);
    };
    auto issue = [&](int slot, int st) __attribute__((always_inline)) { // stage st into slot % NS of the ring
        if (NP == 1 || st < stages_0) issue_of(slot, st, pc[0]);
        else issue_of(slot, st, pc[NP - 1]);
    };

    // ---- queries and the (cos, sin) rows of their positions: through the last slots of the ring, like the tiles and in front
    // of them, so that no load into registers is waited for behind the tiles' (loads complete in order: that would be a wait
    // for the whole ring) ----
    half_t *q_l = smem + (NS - NQ) * 2 * TILE, *cs_l = q_l + Q_HALVES;
    for (int i = wave; i < Q_HALVES / 512; i += W) { // 1 KB: 64 / NC rows, swizzled like a K tile
        const int row = i * (64 / NC) + lane / NC;
        __builtin_amdgcn_global_load_lds(AS_GLOBAL_PTR(q_row(row) + (lane % NC ^ swz(row, NC)) * 8), AS_LDS_PTR(q_l + i * 512), 16, 0, 0);
    }
    for (int i = wave; i < CS_HALVES / 512; i += W) {
        const int row = i * (64 / NCC) + lane / NCC;
        __builtin_amdgcn_global_load_lds(AS_GLOBAL_PTR(cs_row(row) + (lane % NCC ^ (row & (NCC - 1) & 15)) * 4), AS_LDS_PTR(cs_l + i * 512), 16, 0, 0);
    }
    // always NS stages (a short piece's last one more than once): the number of loads in flight is known everywhere
    const int issued = stages > NS ? stages : NS;
#pragma unroll
    for (int st = 0; st < NS - NQ; ++st) issue(st, st < stages ? st : stages - 1);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - NQ) * 2 * LPW) : "memory");
    half8_t qf[HD / 16];
    { // lane (n, hb) takes dims 16 ks + 8 hb .. + 7 of row 32 qt + n
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
    between(qf);

    float16_t o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
    float m_run = -FLT_MAX, l_run = 0.f;
    const float c2 = as_c2<HD>();
    float minus = -1.f;
    asm("" : "+v"(minus)); // not folded: a multiplication, so that conversion, difference and rounding are one instruction
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
        const bool second = NP > 1 && st >= stages_0;
        const int key_st = second ? first_key(st, pc[NP - 1]) : first_key(st, pc[0]);
        const int r_lo = second ? pc[NP - 1].lo : pc[0].lo, r_hi = second ? pc[NP - 1].hi : pc[0].hi;
        // Chunks of 32 keys that the piece begins or ends in: values outside its rows may be anything, NaN included, and
        // become zero in the tile (scores are masked below).
        const int cut_lo = key_st < r_lo ? (r_lo - key_st) & ~31 : SK, cut_hi = key_st + SK > r_hi ? (r_hi - key_st) & ~31 : SK;
        const bool lo_cut = cut_lo < SK && ((r_lo - key_st) & 31), hi_cut = cut_hi < SK && ((r_hi - key_st) & 31);
        if (lo_cut || hi_cut) {
            for (int i = tid; i < HD * 8; i += 64 * W) { // four 16-byte pieces of a dim's row in each of the two chunks
                const int dim = i / 8, at_hi = i / 4 % 2, k0 = (at_hi ? cut_hi : cut_lo) + 8 * (i % 4);
                if (!(at_hi ? hi_cut : lo_cut) || (at_hi && lo_cut && cut_hi == cut_lo)) continue;
                const int f = r_lo - key_st - k0, l = r_hi - key_st - k0; // elements f .. l - 1 stay
                if (f <= 0 && l >= 8) continue;
                half_t *at = vs_ + dim * SK + (k0 / 8 ^ swz(dim, NCV)) * 8;
                half8_t v = load8(at);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e >= f && e < l ? v[e] : (half_t)0.f;
                store8(at, v);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
#pragma unroll
        for (int j = 0; j < S::NCH; ++j) {
            const int kc = 32 * (kg + KG * j), key0 = key_st + kc;   // the chunk in the stage; its first key
            if (key0 >= r_hi || key0 + 32 <= r_lo) continue;        // no key of the piece (the same for every lane)
            float16_t s;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.f;
            const int krow_l = kc + pm;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(load8(ks_ + krow_l * HD + ((2 * ks + hb) ^ swz(krow_l, NC)) * 8), qf[ks], s, 0, 0, 0);
            if (key0 < r_lo || key0 + 32 > r_hi) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = key0 + 16 * (e / 8) + 8 * hb + e % 8;
                    s[e] = key >= r_lo && key < r_hi ? s[e] : -FLT_MAX;
                }
            }
            // The reference of the exponentials lies 7 (in their base 2) below the largest score when it is set and moves when a score
            // leaves it behind by 15, so that O^T is rescaled a handful of times: weights stay below 2^15, inside fp16, and the best ones
            // above 2^7, which leaves 2^-32 of them for the finest step of the type.
            float mx = -FLT_MAX, lo, hi;
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e]);
            xhalf(mx, lo, hi);
            mx = fmaxf(lo, hi);
            if (__builtin_amdgcn_ballot_w64(mx - m_run > 15.f / c2)) {
                const float m_new = mx - m_run > 15.f / c2 ? mx - 7.f / c2 : m_run, alpha = __builtin_amdgcn_exp2f((m_run - m_new) * c2);
                l_run *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
                m_run = m_new;
            }
            // The difference to the reference comes first, then the scaling: with one fused operation on scaled scores every exponent
            // is off by the rounding of the reference, which takes the weights out of fp16 where scores pass 10^7 (and is no
            // faster: 11.6 against 11.2 us at 7 x (1023 + 1), 18.5 and 18.5 at 16 x (8192 + 256)).
            // The operands of the second product are fp16: a weight goes in as the sum of two of them, off by 2^-22 of itself at most,
            // or 2^-25, half the type's finest step.  In one (2^-11) the result was off by 2.4 to 2.9e-4 of its size; the fp16
            // result's own rounding is 2.1e-4.  16 x (8192 + 256) 18.2 -> 18.4 us, 16 x (32768 + 1024)
            // 45.4 -> 46.4, 5 x (5003 + 77) 14.0 -> 14.7.
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f((s[8 * u + e] - m_run) * c2);
                half8_t p, q;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    l_run += w[e] + w[e + 1];
                    half2_t h = {(half_t)w[e], (half_t)w[e + 1]};
                    asm("" : "+v"(h)); // both uses take the converted pair
                    p[e] = h[0];
                    p[e + 1] = h[1];
                    q[e] = (half_t)fmaf((float)h[0], minus, w[e]); // exact before its rounding
                    q[e + 1] = (half_t)fmaf((float)h[1], minus, w[e + 1]);
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const int dim = 32 * (dh * DT + t) + n;
                    const half8_t vf = load8(vs_ + dim * SK + ((kc / 8 + 2 * u + hb) ^ swz(dim, NCV)) * 8);
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p, o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, q, o[t], 0, 0, 0);
                }
            }
        }
        if (st + NS < stages) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); // every wavefront has read the stage
            issue(st, st + NS);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // a short piece's spare loads
    {
        float lo, hi;
        xhalf(l_run, lo, hi);
        l_run = lo + hi;
    }
    // ---- into the LDS, in place of the ring ----
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    float *held = reinterpret_cast<float *>(smem) + wave * as_held<HD, QT, W>();
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4)
            *reinterpret_cast<float4_t *>(held + ((4 * t + e4) * AS_BLOCK + n + AS_HALF * hb) * 4) =
                float4_t{o[t][4 * e4], o[t][4 * e4 + 1], o[t][4 * e4 + 2], o[t][4 * e4 + 3]};
    *reinterpret_cast<float2_t *>(held + 4 * DT * AS_BLOCK * 4 + 2 * lane) = float2_t{m_run, l_run};
    __syncthreads();
}

// What as_tiles left for dims 4 d4 .. + 3 of a query row: the groups of keys joined (unnormalised), the row's reference and sum.
template <int HD, int QT, int W>
__device__ __forceinline__ float4_t as_result(const half_t *smem, int row, int d4, float &m, float &l) {
    using S = AsShape<HD, QT, W>;
    constexpr int PER = as_held<HD, QT, W>();
    // dim 4 d4 = 32 (dh DT + t) + 8 e4 + 4 hb
    const int tile = d4 / 8, dh = tile / S::DT, t = tile % S::DT, e4 = d4 / 2 % 4, n = row % 32;
    const float *base = reinterpret_cast<const float *>(smem) + (row / 32 + QT * S::KG * dh) * PER; // key group 0; the others QT wavefronts apart
    float2_t ml[S::KG];
    m = -FLT_MAX;
#pragma unroll
    for (int g = 0; g < S::KG; ++g) {
        ml[g] = *reinterpret_cast<const float2_t *>(base + g * QT * PER + 4 * S::DT * AS_BLOCK * 4 + 2 * n);
        m = fmaxf(m, ml[g][0]);
    }
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    l = 0.f;
#pragma unroll
    for (int g = 0; g < S::KG; ++g) {
        const float f = __builtin_amdgcn_exp2f((ml[g][0] - m) * as_c2<HD>()); // 0 for a group without a key
        const float4_t x = *reinterpret_cast<const float4_t *>(base + g * QT * PER + ((4 * t + e4) * AS_BLOCK + n + AS_HALF * (d4 % 2)) * 4);
        l += f * ml[g][1];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += f * x[e];
    }
    return o;
}

// One part of the line, left for the merge.
template <int HD, int QT, class QRow, class QSeq, class CsRow>
__device__ __forceinline__ void as_part(half_t *smem, const AsPiece &piece, const int rows, QRow q_row, QSeq q_seq, CsRow cs_row, float *acc,
                                        float *ml) {
    const AsPiece pc[1] = {piece};
    as_tiles<HD, QT, AS_WAVES, 1>(smem, pc, q_row, q_seq, cs_row, [](const half8_t (&)[HD / 16]) {});
    for (int i = threadIdx.x; i < rows * (HD / 4); i += AS_THREADS) {
        const int row = i / (HD / 4), d4 = i % (HD / 4);
        float m, l;
        *reinterpret_cast<float4_t *>(acc + (size_t)i * 4) = as_result<HD, QT, AS_WAVES>(smem, row, d4, m, l);
        if (d4 == 0) *reinterpret_cast<float2_t *>(ml + 2 * row) = float2_t{m, l};
    }
}

// Grid: wgs x KV heads, the KV head fastest: consecutive workgroups go round the XCDs, so that a head's queries and tables stay
// in one XCD's L2.  The arguments in front of `a` are in registers when the kernel starts.
template <int HD, int G, int QT, bool DEV>
__global__ __launch_bounds__(AS_THREADS, AS_WAVES * AS_PER_CU / 4) void attn_shared_part_kernel(float *acc, float *ml, const half_t *qkv,
                                                                                                const float *table, int n_kv_heads, int batch,
                                                                                                int wgs, uint32_t inv, int ldq, int prefix_max,
                                                                                                const SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) half_t smem[];
    const int kvh = blockIdx.x % n_kv_heads, wg = blockIdx.x / n_kv_heads;
    const int rows = batch * G;
    const SharedSeq s0 = shared_seq<DEV>(a, 0); // asked for next to the positions that the line needs
    const AsLine ln = as_line<HD, DEV>(a, n_kv_heads, batch, wgs, inv);
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
        as_part<HD, QT>(smem, AsPiece{s0.kp + (size_t)kvh * prefix_max * HD, s0.vp + (size_t)kvh * HD * prefix_max, prefix_max, from * AS_UNIT,
                                      from * AS_UNIT, end},
                        rows, q_row, q_seq, cs_row, acc + at * HD, ml + at * 2);
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
        as_part<HD, 1>(smem, AsPiece{s.kc + (size_t)kvh * a.max_pos * HD, s.vc + (size_t)kvh * HD * a.max_pos, a.max_pos, b,
                                     b > ln.own_first ? b : ln.own_first, e < end ? e : end},
                       G, q_row, q_seq, cs_row, acc + at * HD, ml + at * 2);
    }
}

// One workgroup per query head and sequence: the parts' weights (first wavefront) and the new token's score (second one) while
// the parts' rows travel, then the weighted sum.  The first head of a group appends the new key and value.  Latency: 4.5 to 6.6 us
// for 32 or 64 heads x 5 to 16 sequences with some 20 to 65 parts each, of which the parts' bytes would take 1 to 3.
#define AS_MERGE_THREADS 256
// parts per thread asked for at once (80 at head size 128, more than a head of eight has)
#define AS_MERGE_AHEAD 10
template <int HD, int G, bool DEV>
__global__ __launch_bounds__(AS_MERGE_THREADS) void attn_shared_merge_kernel(const float *acc, const float *ml, const half_t *qkv, const float *table,
                                                                             int n_kv_heads, int batch, int wgs, uint32_t inv, int ldq, int max_pos,
                                                                             const SharedArgs a) {
    constexpr int LPR = HD / 4, GROUPS = AS_MERGE_THREADS / LPR; // lanes per row of HD floats, rows side by side
    extern __shared__ float weight[]; // one per part
    __shared__ float m_parts, l_parts, m_new;
    __shared__ float4_t part[GROUPS][LPR];
    const int h = blockIdx.x, z = blockIdx.y, kvh = h / G, g = h % G, tid = threadIdx.x, lane = tid % 64;
    const int rows = batch * G, Hq = n_kv_heads * G;
    const float c2 = as_c2<HD>();
    const SharedSeq s = shared_seq<DEV>(a, z);
    const int pos = s.prefix + s.tail, row = s.first + s.tail;
    const AsLine ln = as_line<HD, DEV>(a, n_kv_heads, batch, wgs, inv);
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
            l = l * __builtin_amdgcn_exp2f((M - m) * c2) + p[1] * __builtin_amdgcn_exp2f((p[0] - m) * c2);
            M = m;
            weight[i] = p[0];
        }
        const float all = wave_max(M);
        l = wave_sum(l * __builtin_amdgcn_exp2f((M - all) * c2));
        for (int i = lane; i < ns; i += 64) weight[i] = __builtin_amdgcn_exp2f((weight[i] - all) * c2);
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
        dot = wave_sum(dot);
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
        const float M = fmaxf(m_parts, m_new), f = __builtin_amdgcn_exp2f((m_parts - M) * c2), w = __builtin_amdgcn_exp2f((m_new - M) * c2);
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

// Short lengths: one workgroup of eight wavefronts per KV head and sequence goes through the prefix and the sequence's own rows,
// takes the new token's key with its queries (row G of the query tile: the same position, the same rotation), and writes the
// result -- one launch, the prefix read once per sequence (from the caches of the chip after the first time).
#define AS_DIRECT_WAVES 8
template <int HD, int G, bool DEV>
__global__ __launch_bounds__(64 * AS_DIRECT_WAVES) void attn_shared_direct_kernel(const half_t *qkv, const float *table, half_t *out, int n_kv_heads,
                                                                                 int ldq, int ldo, int prefix_max, int max_pos,
                                                                                 const SharedArgs a) {
    extern __shared__ __attribute__((aligned(16))) half_t smem[];
    __shared__ __attribute__((aligned(16))) half_t k_new[HD], q_rot[G * HD];
    const int kvh = blockIdx.x, z = blockIdx.y, Hq = n_kv_heads * G, tid = threadIdx.x, lane = tid % 64;
    const SharedSeq s = shared_seq<DEV>(a, z);
    const int pos = s.prefix + s.tail;
    const half_t *line = qkv + (size_t)z * ldq, *vn = line + (size_t)(Hq + n_kv_heads + kvh) * HD;
    half_t *kc = s.kc + (size_t)kvh * max_pos * HD, *vc = s.vc + (size_t)kvh * HD * max_pos;
    // dims 4 d4 .. + 3 of head h are this thread's to write (threads beyond the last item: none)
    const int h = tid / (HD / 4), d4 = tid % (HD / 4);
    const half4_t v_new = *reinterpret_cast<const half4_t *>(vn + 4 * d4);
    const AsPiece pc[2] = {{s.kp + (size_t)kvh * prefix_max * HD, s.vp + (size_t)kvh * HD * prefix_max, prefix_max, 0, 0, s.prefix},
                           {kc, vc, max_pos, s.tail > 0 ? s.first & ~7 : 0, s.tail > 0 ? s.first : 0, s.tail > 0 ? s.first + s.tail : 0}};
    auto q_row = [&](int row) { return line + (size_t)(row < G ? kvh * G + row : Hq + kvh) * HD; };
    auto q_seq = [&](int) { return 0; };
    auto cs_row = [&](int) { return table + (size_t)pos * HD; };
    as_tiles<HD, 1, AS_DIRECT_WAVES, 2>(smem, pc, q_row, q_seq, cs_row, [&](const half8_t (&qf)[HD / 16]) {
        const int n = lane % 32, hb = lane / 32;
        if (tid < 64 && n <= G) {
            half_t *d = n < G ? q_rot + n * HD : k_new;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) store8(d + 16 * ks + 8 * hb, qf[ks]);
        }
    });
    static_assert(G * (HD / 4) <= 64 * AS_DIRECT_WAVES, "one item per thread");
    if (tid < G * (HD / 4)) {
        float m, l, dot = 0.f;
        const float4_t o = as_result<HD, 1, AS_DIRECT_WAVES>(smem, h, d4, m, l);
        // the score of the new token: HD / 4 lanes share a head, each a part of the dims
        constexpr int LANES = HD / 4;
        if (d4 < HD / 8) dot = dot8(load8(q_rot + h * HD + 8 * d4), load8(k_new + 8 * d4), 0.f);
#pragma unroll
        for (int x = LANES / 2; x >= 1; x /= 2) dot += __shfl_xor(dot, x);
        const float M = fmaxf(m, dot), f = __builtin_amdgcn_exp2f((m - M) * as_c2<HD>()), w = __builtin_amdgcn_exp2f((dot - M) * as_c2<HD>()), inv = 1.0f / (f * l + w);
        half_t *row = out + (size_t)z * ldo + (size_t)(kvh * G + h) * HD + 4 * d4;
#pragma unroll
        for (int e = 0; e < 4; ++e) row[e] = (half_t)((f * o[e] + w * (float)v_new[e]) * inv);
    }
    // the new key and value into the caches
    if (tid >= 64 * (AS_DIRECT_WAVES - 1)) {
        if (lane < HD / 8) store8(kc + (size_t)(s.first + s.tail) * HD + lane * 8, load8(k_new + lane * 8));
        for (int d = lane; d < HD; d += 64) vc[(size_t)d * max_pos + s.first + s.tail] = vn[d];
    }
}

// Tiles (128 keys at head size 128, 256 at the others) up to which that is faster than two launches, one more at the smaller
// head sizes.  Measured on 1, 4 and 16 sequences, direct against parts: head size 128, four tiles 10.7 / 10.8 / 10.9 against 10.8 /
// 10.9 / 12.9 us, five 12.1 / 12.1 / 12.3 against 10.9 / 10.9 / 13.1; head size 64, five 10.7 / 10.8 / 10.8 against 10.9 / 10.9 / 11.1,
// six 12.0 / 12.0 / 12.1 against 10.9 / 10.9 / 11.0; head size 32, five 8.6 / 8.8 / 8.8 against 10.9 / 10.9 / 11.0.
#define AS_DIRECT_TILES 4
// Workgroups per KV head: two on each of the 256 compute units.
static int as_wgs(int n_kv_heads) { return n_kv_heads < 256 * AS_PER_CU ? 256 * AS_PER_CU / n_kv_heads : 1; }

template <int HD, int G, int QT, bool DEV> static int launch_shared(const SharedArgs &a, const AsPlan &pl, hipStream_t s) {
    const size_t smem = as_lds_bytes<HD, QT, AS_WAVES>() > as_lds_bytes<HD, 1, AS_WAVES>() ? as_lds_bytes<HD, QT, AS_WAVES>() : as_lds_bytes<HD, 1, AS_WAVES>();
    auto kern = attn_shared_part_kernel<HD, G, QT, DEV>;
    static std::atomic<uint64_t> attr_done{0};
    if (smem > 48 * 1024) {
        int rc = llm_ensure_max_smem((const void *)kern, smem, attr_done);
        if (rc != LLM_OK) return rc;
    }
    // no more workgroups than the lengths, or the longest ones that a descriptor may hold, give shares to
    long long used;
    if (DEV) {
        used = ((a.max_prefix + AS_UNIT - 1) / AS_UNIT + (a.max_tail > 0 ? (long long)a.batch * ((a.max_tail + 7 + AS_UNIT - 1) / AS_UNIT + 6) : 0) + 1) / 2;
    } else {
        const int prefix_units = (a.max_prefix + AS_UNIT - 1) / AS_UNIT, lead = (a.host.prefix_len - a.host.row0) & 7;
        int units = 0, tails = 0;
        for (int z = 0; z < a.batch; ++z) {
            const int tail = a.host.seq.pos[z] - a.host.prefix_len;
            units += tail > 0 ? (lead + tail + AS_UNIT - 1) / AS_UNIT : 0;
            tails += tail > 0;
        }
        const AsShare sh = as_share<HD>(prefix_units, units, tails, a.n_kv_heads, pl.wgs, pl.inv);
        used = (prefix_units + units + sh.start * tails + sh.share - 1) / sh.share;
    }
    if (used > pl.wgs) used = pl.wgs;
    if (used > 0) {
        kern<<<dim3((unsigned)used * a.n_kv_heads), dim3(AS_THREADS), smem, s>>>(pl.acc, pl.ml, a.qkv, a.table, a.n_kv_heads, a.batch, pl.wgs,
                                                                                   pl.inv, a.ldq, a.prefix_max, a);
        LLM_LAUNCH_CHECK("attn_shared_part_kernel");
    }
    attn_shared_merge_kernel<HD, G, DEV><<<dim3(a.n_kv_heads * G, a.batch), dim3(AS_MERGE_THREADS), sizeof(float) * 2 * (pl.wgs + 1), s>>>(
        pl.acc, pl.ml, a.qkv, a.table, a.n_kv_heads, a.batch, pl.wgs, pl.inv, a.ldq, a.max_pos, a);
    LLM_LAUNCH_CHECK("attn_shared_merge_kernel");
    return LLM_OK;
}

template <int HD, int G, bool DEV> static int launch_direct(const SharedArgs &a, hipStream_t s) {
    const size_t smem = as_lds_bytes<HD, 1, AS_DIRECT_WAVES>();
    auto kern = attn_shared_direct_kernel<HD, G, DEV>;
    static std::atomic<uint64_t> attr_done{0};
    if (smem > 48 * 1024) {
        int rc = llm_ensure_max_smem((const void *)kern, smem, attr_done);
        if (rc != LLM_OK) return rc;
    }
    kern<<<dim3(a.n_kv_heads, a.batch), dim3(64 * AS_DIRECT_WAVES), smem, s>>>(a.qkv, a.table, a.out, a.n_kv_heads, a.ldq, a.ldo, a.prefix_max, a.max_pos, a);
    LLM_LAUNCH_CHECK("attn_shared_direct_kernel");
    return LLM_OK;
}

template <int HD, int G> static int launch_shared(const SharedArgs &a, void *ws, hipStream_t s) {
    constexpr int SK = AsShape<HD, 1, AS_DIRECT_WAVES>::SK;
    if ((a.max_prefix + SK - 1) / SK + (a.max_tail + SK - 1) / SK <= (HD >= 128 ? AS_DIRECT_TILES : AS_DIRECT_TILES + 1))
        return a.desc ? launch_direct<HD, G, true>(a, s) : launch_direct<HD, G, false>(a, s);
    const int rows = a.batch * G;
    AsPlan pl = {};
    pl.wgs = as_wgs(a.n_kv_heads);
    pl.inv = (uint32_t)(0xffffffffu / pl.wgs + 1);
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
    // Memory in common would make the appended rows race with what is read: none between the own caches, and with the prefix only
    // all of it, both halves, where the new rows lie behind the prefix.
    const size_t per_row = sizeof(half_t) * (size_t)n_kv_heads * head_dim, own_bytes = per_row * max_pos;
    const size_t prefix_bytes = prefix_len > 0 ? per_row * prefix_max_pos : 0;
    for (int z = 0; z < batch; ++z) {
        LLM_REQUIRE(k_caches[z] && v_caches[z] && aligned16(k_caches[z]) && aligned16(v_caches[z]), "%s: cache %d", name, z);
        LLM_REQUIRE(positions[z] >= prefix_len && (long long)positions[z] - row0 < max_pos, "%s: position %d (the prefix has %d, the caches hold %d..%lld)",
                    name, positions[z], prefix_len, row0, (long long)row0 + max_pos - 1);
        auto meets = [&](const void *half, size_t bytes) {
            return bytes > 0 && (ranges_meet(half, bytes, k_caches[z], own_bytes) || ranges_meet(half, bytes, v_caches[z], own_bytes));
        };
        // a prefix inside one of the own caches stays where it is only if row r of that cache is position r
        const bool in_place = k_caches[z] == k_prefix && v_caches[z] == v_prefix && row0 == 0 && prefix_max_pos == max_pos;
        LLM_REQUIRE(in_place || !(meets(k_prefix, prefix_bytes) || meets(v_prefix, prefix_bytes)),
                    "%s: the prefix lies in cache %d, whose row 0 is not position 0, whose size is another or of which it is only a part", name, z);
        LLM_REQUIRE(!ranges_meet(k_caches[z], own_bytes, v_caches[z], own_bytes), "%s: the halves of cache %d overlap", name, z);
        for (int y = 0; y < z; ++y)
            LLM_REQUIRE(!meets(k_caches[y], own_bytes) && !meets(v_caches[y], own_bytes), "%s: sequences %d and %d share a cache", name, y, z);
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
