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

// One workgroup (a wavefront) per sequence and KV head: lane l holds dims of every query head of the group, rows one by one.
template <int HD, int G, bool DEV>
__global__ __launch_bounds__(64) void attn_shared_kernel(const SharedArgs a) {
    const int kvh = blockIdx.x, z = blockIdx.y, lane = threadIdx.x, Hq = a.n_kv_heads * G;
    const SharedSeq s = shared_seq<DEV>(a, z);
    const int pos = s.prefix + s.tail;
    __shared__ __attribute__((aligned(16))) half_t qs[G * HD], kn[HD], vn[HD];
    const half_t *line = a.qkv + (size_t)z * a.ldq;
    const float *cs = a.table + (size_t)pos * HD;
    for (int c = lane; c < (G + 1) * HD / 8; c += 64) { // the group's queries, then the new key
        const int h = c / (HD / 8), e = c % (HD / 8) * 8;
        const half_t *src = line + (h < G ? (size_t)(kvh * G + h) * HD : (size_t)(Hq + kvh) * HD) + e;
        store8((h < G ? qs + h * HD : kn) + e, rope_rotate8(load8(src), cs + e));
    }
    for (int c = lane; c < HD; c += 64) vn[c] = line[(size_t)(Hq + a.n_kv_heads + kvh) * HD + c];
    __syncthreads();
    const int row = s.first + s.tail;
    for (int c = lane; c < HD; c += 64) {
        s.kc[((size_t)kvh * a.max_pos + row) * HD + c] = kn[c];
        s.vc[((size_t)kvh * HD + c) * a.max_pos + row] = vn[c];
    }
    const float scale = 1.0f / sqrtf((float)HD);
    constexpr int DPL = (HD + 63) / 64;
    for (int h = 0; h < G; ++h) {
        float o[DPL] = {}, m = -FLT_MAX, l = 0.f;
        for (int j = 0; j <= pos; ++j) {
            const bool pre = j < s.prefix;
            const int r = pre ? j : s.first + j - s.prefix, stride = pre ? a.prefix_max : a.max_pos;
            const half_t *k = j == pos ? kn : (pre ? s.kp : s.kc) + ((size_t)kvh * stride + r) * HD;
            float dot = 0.f;
            for (int c = lane; c < HD; c += 64) dot += (float)qs[h * HD + c] * (float)k[c];
            const float sc = wave_sum(dot) * scale;
            const float mn = fmaxf(m, sc), alpha = __expf(m - mn), p = __expf(sc - mn);
            m = mn;
            l = l * alpha + p;
            for (int i = 0; i < DPL; ++i) {
                const int c = lane + 64 * i;
                if (c >= HD) continue;
                const float v = j == pos ? (float)vn[c] : (float)(pre ? s.vp : s.vc)[((size_t)kvh * HD + c) * stride + r];
                o[i] = o[i] * alpha + p * v;
            }
        }
        for (int i = 0; i < DPL; ++i)
            if (lane + 64 * i < HD) a.out[(size_t)z * a.ldo + (kvh * G + h) * HD + lane + 64 * i] = (half_t)(o[i] / l);
    }
}

template <int HD, int G> static int launch_shared(const SharedArgs &a, void *ws, hipStream_t s) {
    (void)ws;
    if (a.desc) attn_shared_kernel<HD, G, true><<<dim3(a.n_kv_heads, a.batch), dim3(64), 0, s>>>(a);
    else attn_shared_kernel<HD, G, false><<<dim3(a.n_kv_heads, a.batch), dim3(64), 0, s>>>(a);
    LLM_LAUNCH_CHECK("attn_shared_kernel");
    return LLM_OK;
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
    (void)n_heads, (void)n_kv_heads, (void)head_dim, (void)batch;
    return 16;
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
