"""llm_kv_fork: bits copied as they are, nothing else of the destinations written."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def case(seed, L, Hkv, hd, src_max, dst_max, n_dst):
    rng = np.random.default_rng(seed)
    r = lambda *s: rng.integers(0, 65536, size=s, dtype=np.uint16)  # noqa: E731  any bit pattern, NaN included
    return r(L, Hkv, src_max, hd), r(L, Hkv, hd, src_max), r(n_dst, L, Hkv, dst_max, hd), r(n_dst, L, Hkv, hd, dst_max)


def verify(gpu, c, src_row, dst_row, n):
    k, v, kd, vd = c
    got_k, got_v = gpu.ops.kv_fork(k, v, src_row, kd, vd, dst_row, n)
    want_k, want_v = kd.copy(), vd.copy()
    want_k[:, :, :, dst_row:dst_row + n] = k[None, :, :, src_row:src_row + n]
    want_v[..., dst_row:dst_row + n] = v[None, ..., src_row:src_row + n]
    assert np.array_equal(got_k, want_k) and np.array_equal(got_v, want_v)


@pytest.mark.parametrize("L,Hkv,hd,n_dst", [(1, 1, 8, 1), (3, 2, 32, 2), (2, 8, 128, 16), (2, 3, 64, 5), (1, 5, 40, 3)])
def test_shapes_and_destinations(gpu, L, Hkv, hd, n_dst):
    say("fork", L, Hkv, hd, n_dst)
    verify(gpu, case(1, L, Hkv, hd, 128, 192, n_dst), 0, 0, 100)


@pytest.mark.parametrize("n", [0, 1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 200])
def test_lengths(gpu, n):
    """Every length at offsets that are aligned alike, and not."""
    c = case(2, 2, 2, 32, 256, 256, 2)
    for src_row, dst_row in ((0, 0), (3, 3), (5, 13), (0, 1), (1, 0), (6, 3), (56, 55), (256 - n, 256 - n), (256 - n, 0)):
        verify(gpu, c, src_row, dst_row, n)


@pytest.mark.parametrize("shift", range(-9, 10))
def test_every_relative_alignment(gpu, shift):
    verify(gpu, case(3, 1, 2, 64, 192, 256, 1), 20, 20 + shift, 117)


def test_long_copy(gpu):
    verify(gpu, case(4, 2, 2, 128, 8192, 4096, 2), 4100, 37, 4000)


def test_inside_one_cache(gpu):
    """Ranges of rows of one cache that are apart; they may touch, and share a 16-byte piece of V."""
    k, v, _, _ = case(5, 2, 2, 32, 256, 64, 1)
    for src_row, dst_row, n in ((100, 0, 100), (0, 100, 100), (3, 14, 11), (14, 3, 11), (130, 17, 64), (255, 0, 1)):
        got_k, got_v = gpu.ops.kv_fork(k, v, src_row, None, None, dst_row, n)
        want_k, want_v = k.copy(), v.copy()
        want_k[:, :, dst_row:dst_row + n] = k[:, :, src_row:src_row + n]
        want_v[..., dst_row:dst_row + n] = v[..., src_row:src_row + n]
        assert np.array_equal(got_k[0], want_k) and np.array_equal(got_v[0], want_v)


def test_captured_copy(gpu):
    import ctypes as C
    L, check, ops, Dev = gpu.lib(), gpu.capi.check, gpu.ops, gpu.capi.DevBuf
    k, v, kd, vd = case(6, 2, 2, 64, 128, 128, 2)
    d_k, d_v = Dev.from_host(k), Dev.from_host(v)
    d_ks, d_vs = [Dev.from_host(x) for x in kd], [Dev.from_host(x) for x in vd]
    stream, graph = C.c_void_p(), C.c_void_p()
    check(L.llm_stream_create(C.byref(stream)))
    check(L.llm_graph_capture_begin(stream))
    check(L.llm_kv_fork(d_k.ptr, d_v.ptr, 128, 5, ops._pointers(d_ks), ops._pointers(d_vs), 2, 128, 9, 77, 2, 2, 64, stream))
    check(L.llm_graph_capture_end(stream, C.byref(graph)))
    for rep in range(3):
        k2, v2 = np.roll(k, rep), np.roll(v, rep)
        d_k.upload(k2)
        d_v.upload(v2)
        check(L.llm_graph_launch(graph, stream))
        check(L.llm_stream_sync(stream))
        for i in range(2):
            want_k, want_v = kd[i].copy(), vd[i].copy()
            want_k[:, :, 9:86], want_v[..., 9:86] = k2[:, :, 5:82], v2[..., 5:82]
            assert np.array_equal(d_ks[i].download(), want_k) and np.array_equal(d_vs[i].download(), want_v)
    check(L.llm_graph_destroy(graph))
    check(L.llm_stream_destroy(stream))
