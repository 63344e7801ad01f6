"""llm_logprobs against its definition in 64 bits.

Tolerance, absolute, with y = (x - max) / temperature, p the exact probabilities, u = 2^-24 and D the additions that follow
one another in a sum (a lane of a workgroup of 256 takes at least every 256th logit; the joins of lanes, wavefronts and
workgroups add fewer than 64 more; D = vocab / 256 + 64 also bounds finer splits):
  y: the difference of two fp16 values, times the reciprocal temperature: three roundings, 3 u |y|
  exp(y): the argument's rounding and its product with log2 e, 6 u |y|, and two units of the last place of the result, 4 u
  ln S: the relative error of S, (D + 4 + 6 E|y|) u, one rounding of the logarithm, 2 u (1 + |ln S|)
  log probability: |y| error + ln S error + a rounding of the result
  entropy: ln S error + the relative error of S on E|y| + the same of the second sum, with one product more, 6 E y^2"""
import numpy as np
import pytest

from tests import helpers as H

pytestmark = pytest.mark.gpu

NINF, INF, NAN = 0xfc00, 0x7c00, 0x7e00
U = 2.0 ** -24


def say(*a):
    print(*a, flush=True)


def expected(logits, vocab, ids, k, temperature):
    """(logprob, its tolerance, entropy, its tolerance, top ids, top logprob, its tolerance); logits as bits [rows, ld]."""
    x = H.f16(logits)[:, :vocab] + 0.0
    rows, t = x.shape[0], float(np.float32(temperature))
    n = 0 if ids is None else ids.shape[1]
    lp, lp_tol = np.zeros((rows, n)), np.zeros((rows, n))
    ent, ent_tol = np.zeros(rows), np.zeros(rows)
    ti, tl, tl_tol = np.full((rows, k), -1, np.int32), np.full((rows, k), -np.inf), np.zeros((rows, k))
    depth = vocab / 256 + 64
    for r in range(rows):
        bad = bool(np.any(~(x[r] < np.inf)))
        m = x[r].max() if not bad else 0.0
        with np.errstate(invalid="ignore"):
            y = (x[r] - (m if np.isfinite(m) else 0.0)) / t
        if bad:
            lp[r], ent[r], tl[r] = np.nan, np.nan, np.nan
            continue
        s = np.exp(y).sum()
        p = np.exp(y) / s if s else np.zeros(vocab)
        fin = np.isfinite(y)
        ey, eyy = (p[fin] * np.abs(y[fin])).sum(), (p[fin] * y[fin] ** 2).sum()
        ls = np.log(s) if s else 0.0
        e_s = (depth + 4 + 6 * ey) * U
        e_ls = e_s + 2 * U * (1 + abs(ls))
        logp = y - ls
        tol = np.where(fin, 3 * U * np.abs(np.where(fin, y, 0)) + e_ls + 2 * U * np.abs(np.where(fin, logp, 0)), 0)
        ent[r] = ls + ey if s else 0.0
        ent_tol[r] = e_ls + e_s * ey + (depth + 8) * U * ey + 6 * U * eyy + 2 * U * abs(ent[r])
        if n:
            ok = (ids[r] >= 0) & (ids[r] < vocab)
            at = np.where(ok, ids[r], 0)
            lp[r], lp_tol[r] = np.where(ok, logp[at], np.nan), tol[at]
        order = np.lexsort((np.arange(vocab), -x[r]))[:k]
        order = order[np.isfinite(x[r][order])]
        ti[r, :order.size], tl[r, :order.size], tl_tol[r, :order.size] = order, logp[order], tol[order]
    return lp, lp_tol, ent, ent_tol, ti, tl, tl_tol


def close(got, want, tol):
    with np.errstate(invalid="ignore"):
        same = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got.astype(np.float64) - want) <= tol)
    fin = np.isfinite(want) & np.isfinite(got)
    if fin.any():
        say("  worst error / tolerance: %.3f" % float(np.max(np.abs(got[fin] - want[fin]) / np.maximum(tol[fin], 1e-300))))
    return bool(same.all())


def verify(gpu, logits, vocab=None, ids=None, k=0, temperature=1.0, **kw):
    vocab = logits.shape[1] if vocab is None else vocab
    lp, lp_tol, ent, ent_tol, ti, tl, tl_tol = expected(logits, vocab, ids, k, temperature)
    g_lp, g_ent, g_ti, g_tl = gpu.ops.logprobs(logits, vocab, ids, k, temperature, **kw)
    assert close(g_lp, lp, lp_tol)
    assert close(g_ent, ent, ent_tol)
    assert np.array_equal(g_ti, ti)
    assert close(g_tl, tl, tl_tol)


def rows_of(seed, rows, ld, scale=2.5):
    rng = np.random.default_rng(seed)
    x = H.bits(rng.standard_normal((rows, ld)) * scale)
    ids = rng.integers(0, ld, size=(rows, 3)).astype(np.int32)
    return x, ids


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 64, 65, 255, 256, 257, 1000, 2047, 2048, 2049, 4096, 16384, 16385, 32003, 128256, 131072])
def test_vocabularies(gpu, vocab):
    rows = 3 if vocab < 20000 else 2
    x, ids = rows_of(vocab, rows, vocab)
    say("vocab", vocab)
    verify(gpu, x, ids=ids, k=min(20, vocab))


@pytest.mark.parametrize("rows", [1, 2, 3, 16, 37, 257, 600, 5000])
def test_row_counts(gpu, rows):
    x, ids = rows_of(rows, rows, 1003)
    say("rows", rows)
    verify(gpu, x, ids=ids, k=4)


@pytest.mark.parametrize("k", [0, 1, 2, 5, 19, 31, 32])
@pytest.mark.parametrize("vocab", [32, 515, 70001])
def test_top_counts(gpu, k, vocab):
    x, ids = rows_of(k, 2, vocab)
    verify(gpu, x, ids=ids, k=k)


@pytest.mark.parametrize("n_ids", [0, 1, 2, 16])
def test_given_tokens(gpu, n_ids):
    x, _ = rows_of(1, 5, 4096)
    ids = np.random.default_rng(2).integers(0, 4096, size=(5, n_ids)).astype(np.int32)
    if n_ids:
        ids[0, 0], ids[1, -1], ids[2, 0], ids[3, 0], ids[4, -1] = -1, 4096, 2 ** 31 - 1, -2 ** 31, 4095
    verify(gpu, x, ids=ids, k=3)
    if n_ids > 1:
        ids[:] = 77  # the same token several times
        verify(gpu, x, ids=ids)


@pytest.mark.parametrize("offset", range(9))
@pytest.mark.parametrize("pad", [0, 1, 5, 8])
def test_rows_that_start_anywhere(gpu, offset, pad):
    """Columns behind the vocabulary are +inf and would spoil every value if they were read as logits."""
    x, ids = rows_of(offset, 4, 777 + pad)
    x[:, 777:] = INF
    verify(gpu, x, 777, ids % 777, 6, offset=offset)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 1.9, 40.0])
def test_temperatures(gpu, temperature):
    x, ids = rows_of(3, 4, 5000)
    verify(gpu, x, ids=ids, k=7, temperature=temperature)


def test_ties_go_to_the_lowest_index(gpu):
    for vocab in (64, 4096, 40000):
        x = np.full((4, vocab), H.bits(1.0), np.uint16)
        x[1] = H.bits((np.arange(vocab) % 3).astype(np.float32))         # a third of the row at the maximum
        x[2, ::2] = 0x8000                                                # -0 and +0 are equal
        x[2, 1::2] = 0
        x[3] = H.bits(-(np.arange(vocab) // 7 % 50).astype(np.float32))
        verify(gpu, x, ids=np.array([[0], [1], [2], [3]], np.int32), k=32)


def test_sorted_rows(gpu):
    """Ascending and descending logits: the best are all at one end of the row, next to one another."""
    ramp = H.bits(np.linspace(-20, 20, 30000).astype(np.float32))
    verify(gpu, np.stack([ramp, ramp[::-1]]), ids=np.array([[0], [29999]], np.int32), k=32)


@pytest.mark.parametrize("left", [0, 1, 2, 31, 33, 500])
def test_masked_rows(gpu, left):
    """All but `left` logits are -inf, the type's lowest value, or both, scattered and in one run."""
    for vocab in (600, 20000):
        x, ids = rows_of(left, 6, vocab)
        rng = np.random.default_rng(left)
        for r in range(6):
            keep = rng.permutation(vocab)[:left] if r % 2 else np.arange(left) + min(vocab // 3, vocab - left)
            row = np.full(vocab, NINF if r < 4 else 0xfbff, np.uint16)
            if r == 5:
                row[: vocab // 2] = NINF
            row[keep] = x[r, keep]
            x[r] = row
            if left:
                ids[r, 0] = keep[0]
        verify(gpu, x, ids=ids, k=32)


def test_lowest_value_only(gpu):
    """Every logit at the type's lowest value is a uniform distribution; with -inf among them they share all probability."""
    x = np.full((3, 3000), 0xfbff, np.uint16)
    x[1, 5:] = NINF
    x[2, 1::2] = NINF
    verify(gpu, x, ids=np.array([[0, 9], [4, 5], [1, 2]], np.int32), k=6)


def test_rows_without_a_distribution(gpu):
    """NaN (either sign) and +inf anywhere spoil their row, and only theirs."""
    x, ids = rows_of(9, 8, 18000)
    x[1, 0], x[2, 17999], x[3, 9000], x[4, 123] = NAN, 0xfe00, INF, 0x7c01
    x[5] = NINF
    x[5, 77] = NAN
    x[6] = INF
    verify(gpu, x, ids=ids, k=5)


def test_extremes_of_the_range(gpu):
    x = np.zeros((2, 4097), np.uint16)
    x[0] = 0xfbff
    x[0, 4096] = 0x7bff  # 65504 against -65504
    x[1, 7] = 0x0001     # a subnormal above zeros
    verify(gpu, x, ids=np.array([[4096, 0], [7, 0]], np.int32), k=4)


def test_one_workspace_for_calls_of_other_shapes(gpu):
    shapes = [(1, 128256, 20), (700, 300, 3), (16, 40000, 32), (5000, 64, 1), (3, 128256, 0)]
    size = max(gpu.lib().llm_logprobs_workspace_bytes(*s) for s in shapes)
    ws = gpu.ops._zeroed(size)
    for rows, vocab, k in shapes + shapes[::-1]:
        x, ids = rows_of(rows, rows, vocab)
        a = gpu.ops.logprobs(x, ids=ids, k=k, ws=ws, repeats=2)
        b = gpu.ops.logprobs(x, ids=ids, k=k)
        assert all(np.array_equal(p.view(np.uint32), q.view(np.uint32)) for p, q in zip(a, b)), (rows, vocab, k)


def test_captured_call(gpu):
    import ctypes as C
    L, check, ops, Dev = gpu.lib(), gpu.capi.check, gpu.ops, gpu.capi.DevBuf
    x, ids = rows_of(4, 5, 50000)
    d_x, d_i = Dev.from_host(x), Dev.from_host(ids)
    d_lp, d_h, d_ti, d_tl = Dev((5, 3), np.float32), Dev((5,), np.float32), Dev((5, 8), np.int32), Dev((5, 8), np.float32)
    ws = ops._zeroed(L.llm_logprobs_workspace_bytes(5, 50000, 8))
    stream, graph = C.c_void_p(), C.c_void_p()
    check(L.llm_stream_create(C.byref(stream)))
    check(L.llm_graph_capture_begin(stream))
    check(L.llm_logprobs(d_x.ptr, 50000, 5, 50000, 0.7, d_i.ptr, 3, d_lp.ptr, d_h.ptr, 8, d_ti.ptr, d_tl.ptr, ws.ptr, stream))
    check(L.llm_graph_capture_end(stream, C.byref(graph)))
    for rep in range(4):
        y = np.roll(x, 1000 * rep, 1)
        d_x.upload(y)
        check(L.llm_graph_launch(graph, stream))
        check(L.llm_stream_sync(stream))
        eager = ops.logprobs(y, ids=ids, k=8, temperature=0.7)
        for got, want in zip((d_lp, d_h, d_ti, d_tl), eager):
            assert np.array_equal(got.download().view(np.uint32), want.view(np.uint32)), rep
    check(L.llm_graph_destroy(graph))
    check(L.llm_stream_destroy(stream))


def test_a_workspace_for_many_rows_holds_a_call_of_fewer(gpu):
    """511 rows are cut into two chunks each where 512 are not: the same workspace, and nothing is written behind it."""
    vocab, k = 9000, 32
    size = gpu.lib().llm_logprobs_workspace_bytes(512, vocab, k)
    guard = 1 << 20
    ws = gpu.capi.DevBuf((size + guard,), np.uint8)
    mark = np.concatenate([np.zeros(size, np.uint8), np.full(guard, 0xa5, np.uint8)])
    for rows in (512, 511, 256, 255, 8, 1):
        x, ids = rows_of(rows, rows, vocab)
        ws.upload(mark)
        a = gpu.ops.logprobs(x, ids=ids, k=k, ws=ws)
        assert np.all(ws.download()[size:] == 0xa5), rows
        b = gpu.ops.logprobs(x, ids=ids, k=k)
        assert all(np.array_equal(p.view(np.uint32), q.view(np.uint32)) for p, q in zip(a, b)), rows


@pytest.mark.parametrize("temperature", [1e-30, 1e-20, 1e-12, 1e-10, 1e-9, 1e-8, 1e-6, 1e-5, 1e-3, 1e-2, 1e4, 1e30, 3.4e38])
@pytest.mark.parametrize("vocab", [2, 1003, 70001])
def test_temperatures_over_the_accepted_range(gpu, temperature, vocab):
    """Maxima whose products with the reciprocal temperature are rounded, from the smallest logits to the largest; rows with two
    equal maxima, with a mask, and of one magnitude throughout."""
    peaks = [6.30, 12.5, 13.25, 14.3, 39.9, 65504.0, -65504.0, 6e-8, 0.333, -7.77]
    x, _ = rows_of(17, 2 * len(peaks), vocab)
    ids = np.zeros((2 * len(peaks), 2), np.int32)
    for r, peak in enumerate(peaks):
        for row in (r, r + len(peaks)):
            top = H.bits(peak).item()
            x[row] = H.bits(np.maximum(np.minimum(H.f16(x[row]), peak - abs(peak) * 2.0 ** -9), -65504.0))
            x[row, vocab // 3] = top
            ids[row] = vocab // 3, vocab - 1
        x[r + len(peaks), vocab - 1] = top   # the second of two equal ones
        x[r, : vocab // 4] = NINF
    say("temperature", temperature, "vocab", vocab)
    verify(gpu, x, ids=ids, k=min(vocab, 5), temperature=temperature)


def test_entropy_is_never_negative(gpu):
    """Rows with one logit ahead by anything from nothing to all: ln S and the mean that is taken from it are rounded apart."""
    for vocab in (2, 50, 5000):
        rng = np.random.default_rng(vocab)
        x = H.bits(rng.standard_normal((400, vocab)))
        x[:, 0] = H.bits(np.linspace(3, 40, 400))
        for t in (1e-8, 1e-3, 0.3, 1.0, 2.0):
            _, ent, _, _ = gpu.ops.logprobs(x, temperature=t)
            say("vocab", vocab, "temperature", t, "least", ent.min())
            assert ent.min() >= 0.0
        verify(gpu, x[::40])
