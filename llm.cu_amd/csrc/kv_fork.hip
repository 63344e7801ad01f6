// Rows of a KV cache copied into the caches of other sequences, all layers and both halves in one launch.
#include "common.hpp"
#include "ranges.hpp"

#define KF_MAX_DST LLM_MAX_BATCH
#define KF_THREADS 256
#define KF_NT_ROWS 256 // rows from which V is stored with NT_V

struct KfArgs {
    const half_t *k_src, *v_src;
    half_t *k_dst[KF_MAX_DST], *v_dst[KF_MAX_DST];
    int n_dst, src_max, dst_max, src_row, dst_row, n, head_dim;
    int k_parts, row_parts; // workgroups per head for K; per group of V's dims
    int lanes_log2;         // lanes per dim of V
};

// eight halves from any element: one 16-byte load, which the memory pipeline takes at any 2-byte address
__device__ __forceinline__ half8_t load8_any(const half_t *p) {
    half8_t v;
    __builtin_memcpy(&v, p, sizeof v);
    return v;
}

__device__ __forceinline__ void store8_nt(half_t *p, half8_t v) { // without keeping the line
    __builtin_nontemporal_store(__builtin_bit_cast(uint4_t, v), reinterpret_cast<uint4_t *>(p));
}

// Grid (parts of a head's K + parts of its V, layers * kv heads); a thread takes one 16-byte chunk, aligned at the destination,
// and stores it to every destination.  K is one contiguous piece per head, V a piece per dim, whose first and last few rows
// (those that do not fill a chunk) are dealt to the dim's lanes one by one.
// Bound by the memory: 2048 rows of an 8B cache (268 MB) to four destinations 263 us, 5.1 TB/s read and written (a plain copy
// of that size: 5.1); 1000 rows whose offsets differ by an odd number 45 us, 5.8 TB/s.  One chunk per thread: with two, short
// pieces lack wavefronts (33 rows to two destinations 12.9 against 7.9 us).  Pieces of a few hundred bytes pay for the lines
// they share with rows that stay (200 rows to eight destinations: 3.3 TB/s).
// NT_V: V's chunks stored without keeping their lines (K's always are) -- for long pieces (1000 rows: 45 against 52 us); the end
// lines of short ones are joined in the L2 when they are kept (100 rows to four destinations: 17.6 against 42 us; 200 rows
// to eight: 71 against 69 us).
template <bool NT_V> __global__ __launch_bounds__(KF_THREADS) void kv_fork_kernel(const KfArgs a) {
    const size_t head = blockIdx.y;
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < a.k_parts) {
        const size_t c = (size_t)blockIdx.x * KF_THREADS + tid;
        if (c * 8 >= (size_t)a.n * a.head_dim) return;
        const half8_t v = load8_nt(a.k_src + (head * a.src_max + a.src_row) * a.head_dim + c * 8);
        const size_t d = (head * a.dst_max + a.dst_row) * a.head_dim + c * 8;
        for (int i = 0; i < a.n_dst; ++i) store8_nt(a.k_dst[i] + d, v);
        return;
    }
    const int lanes = 1 << a.lanes_log2, part = blockIdx.x - a.k_parts, l = tid & (lanes - 1);
    const int dim = part / a.row_parts * (KF_THREADS >> a.lanes_log2) + (tid >> a.lanes_log2), row_part = part % a.row_parts;
    if (dim >= a.head_dim) return;
    const int last = a.dst_row + a.n, shift = a.src_row - a.dst_row; // destination row r gets source row r + shift
    const half_t *src = a.v_src + (head * a.head_dim + dim) * a.src_max;
    const size_t d = (head * a.head_dim + dim) * a.dst_max;
    const int r = ((a.dst_row + 7) & ~7) + 8 * (row_part * lanes + l);
    if (r + 8 <= last) {
        const half8_t v = load8_any(src + (r + shift));
        for (int i = 0; i < a.n_dst; ++i) {
            if (NT_V) store8_nt(a.v_dst[i] + d + r, v);
            else store8(a.v_dst[i] + d + r, v);
        }
    }
    if (row_part == 0) {
        int front = -a.dst_row & 7, back = last & 7; // rows in front of the first chunk, behind the last one
        if (front + back > a.n || front > a.n) { // the range lies inside one chunk, or touches two and fills none
            front = a.n;
            back = 0;
        }
        for (int e = l; e < front + back; e += lanes) {
            const int q = e < front ? a.dst_row + e : last - back + (e - front);
            const half_t v = src[q + shift];
            for (int i = 0; i < a.n_dst; ++i) a.v_dst[i][d + q] = v;
        }
    }
}

extern "C" int llm_kv_fork(const uint16_t *k_src, const uint16_t *v_src, int src_max_pos, int src_row, uint16_t *const *k_dsts,
                           uint16_t *const *v_dsts, int n_dst, int dst_max_pos, int dst_row, int n_rows, int n_layers,
                           int n_kv_heads, int head_dim, llm_stream_t stream) {
    LLM_REQUIRE(k_src && v_src && k_dsts && v_dsts, "llm_kv_fork: null pointer");
    LLM_REQUIRE(n_dst >= 1 && n_dst <= KF_MAX_DST, "llm_kv_fork: %d destinations (1..%d)", n_dst, KF_MAX_DST);
    LLM_REQUIRE(n_layers >= 1 && n_kv_heads >= 1 && (long long)n_layers * n_kv_heads <= 65535,
                "llm_kv_fork: %d layers of %d kv heads (at most 65535 together)", n_layers, n_kv_heads);
    LLM_REQUIRE(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 1024, "llm_kv_fork: head_dim=%d (a multiple of 8 up to 1024)", head_dim);
    LLM_REQUIRE(src_max_pos > 0 && src_max_pos % 64 == 0 && dst_max_pos > 0 && dst_max_pos % 64 == 0,
                "llm_kv_fork: max_pos %d -> %d must be multiples of 64", src_max_pos, dst_max_pos);
    LLM_REQUIRE(src_max_pos <= 1 << 30 && dst_max_pos <= 1 << 30, "llm_kv_fork: max_pos %d -> %d (at most 2^30)", src_max_pos, dst_max_pos);
    LLM_REQUIRE(n_rows >= 0 && src_row >= 0 && src_row <= src_max_pos && n_rows <= src_max_pos - src_row,
                "llm_kv_fork: %d rows from row %d of %d", n_rows, src_row, src_max_pos);
    LLM_REQUIRE(dst_row >= 0 && dst_row <= dst_max_pos && n_rows <= dst_max_pos - dst_row, "llm_kv_fork: %d rows to row %d of %d",
                n_rows, dst_row, dst_max_pos);
    LLM_REQUIRE(aligned16(k_src) && aligned16(v_src), "llm_kv_fork: caches must be 16-byte aligned");
    KfArgs a = {};
    a.k_src = (const half_t *)k_src;
    a.v_src = (const half_t *)v_src;
    a.n_dst = n_dst;
    a.src_max = src_max_pos;
    a.dst_max = dst_max_pos;
    a.src_row = src_row;
    a.dst_row = dst_row;
    a.n = n_rows;
    a.head_dim = head_dim;
    const size_t per_row = sizeof(half_t) * (size_t)n_layers * n_kv_heads * head_dim;
    const size_t src_bytes = per_row * src_max_pos, dst_bytes = per_row * dst_max_pos;
    const bool rows_apart = src_row + n_rows <= dst_row || dst_row + n_rows <= src_row;
    const void *bufs[2 * KF_MAX_DST];
    for (int i = 0; i < n_dst; ++i) {
        LLM_REQUIRE(k_dsts[i] && v_dsts[i] && aligned16(k_dsts[i]) && aligned16(v_dsts[i]), "llm_kv_fork: destination %d", i);
        a.k_dst[i] = (half_t *)k_dsts[i];
        a.v_dst[i] = (half_t *)v_dsts[i];
        bufs[2 * i] = k_dsts[i];
        bufs[2 * i + 1] = v_dsts[i];
    }
    // A destination may be the source cache itself when the two ranges of rows are apart; any other memory in common
    // (another offset into it, K on V, one destination twice) would make the copies race with one another.
    for (int i = 0; i < 2 * n_dst; ++i) {
        const bool k_half = i % 2 == 0;
        const void *same = k_half ? (const void *)k_src : (const void *)v_src, *other = k_half ? (const void *)v_src : (const void *)k_src;
        const bool in_place = bufs[i] == same && src_max_pos == dst_max_pos && rows_apart;
        LLM_REQUIRE(in_place || !ranges_meet(bufs[i], dst_bytes, same, src_bytes),
                    "llm_kv_fork: destination %d overlaps the source (the same cache takes ranges of rows that are apart)", i / 2);
        LLM_REQUIRE(!ranges_meet(bufs[i], dst_bytes, other, src_bytes), "llm_kv_fork: destination %d overlaps the source's other half", i / 2);
        for (int j = 0; j < i; ++j)
            LLM_REQUIRE(!ranges_meet(bufs[i], dst_bytes, bufs[j], dst_bytes), "llm_kv_fork: destinations %d and %d overlap", j / 2, i / 2);
    }
    if (n_rows == 0) return LLM_OK;
    const size_t k_chunks = (size_t)n_rows * head_dim / 8;
    const int v_chunks = ((dst_row + n_rows) >> 3) - ((dst_row + 7) >> 3); // full ones; not positive when the range fills none
    a.lanes_log2 = 3;
    while (a.lanes_log2 < 6 && (1 << a.lanes_log2) < v_chunks) ++a.lanes_log2;
    const int lanes = 1 << a.lanes_log2, dims = KF_THREADS / lanes;
    a.k_parts = (int)((k_chunks + KF_THREADS - 1) / KF_THREADS);
    a.row_parts = v_chunks > lanes ? (v_chunks + lanes - 1) / lanes : 1;
    const unsigned v_parts = (unsigned)((head_dim + dims - 1) / dims) * a.row_parts;
    const dim3 grid(a.k_parts + v_parts, (unsigned)(n_layers * n_kv_heads));
    if (n_rows >= KF_NT_ROWS) kv_fork_kernel<true><<<grid, dim3(KF_THREADS), 0, (hipStream_t)stream>>>(a);
    else kv_fork_kernel<false><<<grid, dim3(KF_THREADS), 0, (hipStream_t)stream>>>(a);
    LLM_LAUNCH_CHECK("kv_fork_kernel");
    return LLM_OK;
}
