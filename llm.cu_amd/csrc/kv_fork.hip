// Rows of a KV cache copied into the caches of other sequences, all layers and both halves in one launch.
#include "common.hpp"

#define KF_MAX_DST LLM_MAX_BATCH
#define KF_THREADS 256

struct KfArgs {
    const half_t *k_src, *v_src;
    half_t *k_dst[KF_MAX_DST], *v_dst[KF_MAX_DST];
    int n_dst, src_max, dst_max, src_row, dst_row, n, head_dim;
};

// Grid (parts, layers * kv heads, 2): z = 0 copies K (one contiguous piece per head), z = 1 V (a piece per dim).
__global__ __launch_bounds__(KF_THREADS) void kv_fork_kernel(const KfArgs a) {
    const size_t head = blockIdx.y;
    const size_t step = (size_t)gridDim.x * KF_THREADS;
    if (blockIdx.z == 0) {
        const size_t s0 = (head * a.src_max + a.src_row) * a.head_dim, d0 = (head * a.dst_max + a.dst_row) * a.head_dim;
        const size_t chunks = (size_t)a.n * a.head_dim / 8;
        for (size_t c = (size_t)blockIdx.x * KF_THREADS + threadIdx.x; c < chunks; c += step) {
            const half8_t v = load8(a.k_src + s0 + c * 8);
            for (int i = 0; i < a.n_dst; ++i) store8(a.k_dst[i] + d0 + c * 8, v);
        }
    } else {
        const size_t s0 = head * a.head_dim * a.src_max + a.src_row, d0 = head * a.head_dim * a.dst_max + a.dst_row;
        const size_t total = (size_t)a.n * a.head_dim;
        for (size_t c = (size_t)blockIdx.x * KF_THREADS + threadIdx.x; c < total; c += step) {
            const size_t dim = c / a.n, row = c % a.n;
            const half_t v = a.v_src[s0 + dim * a.src_max + row];
            for (int i = 0; i < a.n_dst; ++i) a.v_dst[i][d0 + dim * a.dst_max + row] = v;
        }
    }
}

static bool ranges_meet(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + b_bytes && y < x + a_bytes;
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
    const size_t elems = (size_t)n_rows * head_dim;
    size_t parts = (elems + KF_THREADS * 8 - 1) / (KF_THREADS * 8);
    if (parts > 64) parts = 64;
    kv_fork_kernel<<<dim3((unsigned)parts, (unsigned)(n_layers * n_kv_heads), 2), dim3(KF_THREADS), 0, (hipStream_t)stream>>>(a);
    LLM_LAUNCH_CHECK("kv_fork_kernel");
    return LLM_OK;
}
