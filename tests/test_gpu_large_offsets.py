"""Cache forks, shared-prefix attention and log probabilities where byte offsets pass 32 bits: large buffers of which only the
places that a result depends on are written (the others may hold anything)."""
import ctypes as C

import numpy as np
import pytest

from tests import helpers as H
from tests import test_gpu_attn_shared as shared_tests
from tests import test_gpu_logprobs as logprob_tests

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


class Large:
    """fp16 device memory written and read in pieces at element offsets."""

    def __init__(self, gpu, elems):
        self.gpu, self.buf = gpu, gpu.capi.DevBuf((elems,), np.uint16)
        self.ptr = self.buf.ptr

    def put(self, at, a):
        a = np.ascontiguousarray(a, dtype=np.uint16)
        assert 0 <= at and at + a.size <= self.buf.shape[0]
        self.gpu.capi.check(self.gpu.lib().llm_memcpy_h2d(self.ptr + 2 * at, a.ctypes.data, a.nbytes, None))

    def get(self, at, n):
        assert 0 <= at and at + n <= self.buf.shape[0]
        out = np.empty(n, np.uint16)
        self.gpu.capi.check(self.gpu.lib().llm_memcpy_d2h(out.ctypes.data, self.ptr + 2 * at, out.nbytes, None))
        return out


def test_log_probabilities_of_many_rows(gpu):
    """Rows 0 .. 19999 of 128256 logits: 5.1 GB; the first one, one beyond 2^32 bytes, and the last one."""
    rows, vocab = 20000, 128256
    x, ids = logprob_tests.rows_of(9, 3, vocab)
    at = [0, 2 ** 31 // vocab + 1, rows - 1]
    big = Large(gpu, rows * vocab)
    for r, line in zip(at, x):
        big.put(r * vocab, line)
    given = np.zeros((rows, 3), np.int32)
    given[at] = ids
    Dev, L = gpu.capi.DevBuf, gpu.lib()
    d_i = Dev.from_host(given)
    d_lp, d_h, d_ti, d_tl = Dev((rows, 3), np.float32), Dev((rows,), np.float32), Dev((rows, 4), np.int32), Dev((rows, 4), np.float32)
    ws = gpu.ops._zeroed(L.llm_logprobs_workspace_bytes(rows, vocab, 4))
    say("log probabilities of", rows, "rows")
    gpu.capi.check(L.llm_logprobs(big.ptr, vocab, rows, vocab, 1.0, d_i.ptr, 3, d_lp.ptr, d_h.ptr, 4, d_ti.ptr, d_tl.ptr, ws.ptr, None))
    lp, lp_tol, ent, ent_tol, ti, tl, tl_tol = logprob_tests.expected(x, vocab, ids, 4, 1.0)
    assert logprob_tests.close(d_lp.download()[at], lp, lp_tol) and logprob_tests.close(d_h.download()[at], ent, ent_tol)
    assert np.array_equal(d_ti.download()[at], ti) and logprob_tests.close(d_tl.download()[at], tl, tl_tol)


def test_fork_of_a_large_cache(gpu):
    """Five heads of 128 x 2^22 positions: 1 GB a head; rows near the end of every head go to the front of a small cache, and back."""
    heads, hd, big_max, small_max, n = 5, 128, 1 << 22, 256, 101
    rng = np.random.default_rng(4)
    k, v = H.bits(rng.standard_normal((heads, n, hd))), H.bits(rng.standard_normal((heads, hd, n)))
    big_k, big_v = Large(gpu, heads * big_max * hd), Large(gpu, heads * big_max * hd)
    small_k, small_v = Large(gpu, heads * small_max * hd), Large(gpu, heads * small_max * hd)
    src = big_max - n - 3
    for h in range(heads):
        big_k.put((h * big_max + src) * hd, k[h])
        for d in range(hd):
            big_v.put((h * hd + d) * big_max + src, v[h, d])
    one = lambda b: (C.c_void_p * 1)(b.ptr)  # noqa: E731
    fork = gpu.lib().llm_kv_fork
    say("fork of a large cache")
    gpu.capi.check(fork(big_k.ptr, big_v.ptr, big_max, src, one(small_k), one(small_v), 1, small_max, 6, n, 1, heads, hd, None))
    for h in range(heads):
        assert np.array_equal(small_k.get((h * small_max + 6) * hd, n * hd).reshape(n, hd), k[h])
        assert np.array_equal(np.stack([small_v.get((h * hd + d) * small_max + 6, n) for d in range(hd)]), v[h])
    back = big_max - 2 * n - 50
    gpu.capi.check(fork(small_k.ptr, small_v.ptr, small_max, 6, one(big_k), one(big_v), 1, big_max, back, n, 1, heads, hd, None))
    for h in range(heads):
        assert np.array_equal(big_k.get((h * big_max + back) * hd, n * hd).reshape(n, hd), k[h])
        for d in (0, 1, hd - 1):
            assert np.array_equal(big_v.get((h * hd + d) * big_max + back, n), v[h, d])
            assert np.array_equal(big_v.get((h * hd + d) * big_max + src, n), v[h, d])  # what was there stays


@pytest.mark.parametrize("prefix", [200, 1500])
def test_shared_attention_in_large_caches(gpu, prefix):
    """The prefix in a cache of 2^22 positions, the answers in caches of 2^21, five heads of 128: one launch and two."""
    heads, hd, pmax, max_pos, B = 5, 128, 1 << 22, 1 << 21, 2
    c = shared_tests.case(31, B, prefix, [3, 70], (heads, heads, hd), True)
    small = c["kcs"].shape[2]
    Dev, L = gpu.capi.DevBuf, gpu.lib()
    kp, vp = Large(gpu, heads * pmax * hd), Large(gpu, heads * pmax * hd)
    ks, vs = [[Large(gpu, heads * max_pos * hd) for _ in range(B)] for _ in range(2)]
    for h in range(heads):
        kp.put(h * pmax * hd, c["kp"][h])
        for d in range(hd):
            vp.put((h * hd + d) * pmax, c["vp"][h, d])
        for z in range(B):
            ks[z].put(h * max_pos * hd, c["kcs"][z, h])
            for d in range(hd):
                vs[z].put((h * hd + d) * max_pos, c["vcs"][z, h, d])
    d_q, d_t = Dev.from_host(c["qkv"]), Dev.from_host(gpu.ops.rope_table(prefix + small, hd))
    d_o, ws = Dev((B, heads * hd), np.uint16), gpu.ops._zeroed(L.llm_attn_shared_workspace_bytes(heads, heads, hd, B))
    ptrs = lambda bufs: (C.c_void_p * B)(*[b.ptr for b in bufs])  # noqa: E731
    say("shared attention in large caches, prefix", prefix)
    gpu.capi.check(L.llm_attn_decode_rope_shared(d_q.ptr, 3 * heads * hd, kp.ptr, vp.ptr, prefix, pmax, ptrs(ks), ptrs(vs),
                                                 (C.c_int * B)(*c["positions"]), prefix, B, d_o.ptr, heads * hd, d_t.ptr, heads, heads,
                                                 hd, max_pos, ws.ptr, None))
    out = d_o.download()
    got_k, got_v = c["kcs"].copy(), c["vcs"].copy()
    for z in range(B):
        for h in range(heads):
            got_k[z, h] = ks[z].get(h * max_pos * hd, small * hd).reshape(small, hd)
            got_v[z, h] = np.stack([vs[z].get((h * hd + d) * max_pos, small) for d in range(hd)])
    shared_tests.verify((out, got_k, got_v), shared_tests.expected(c))
