"""llm_attn_decode_rope_shared and its descriptor form against the attention of every sequence on its own in 64 bits.

Tolerance, per output element, with w the exact softmax weights and n the positions:
  half an fp16 step of the result                                          2^-11 |o|
  the weights rounded to fp16 for the second product                      2^-11 sum w |v|;
      a weight below the normal fp16 range is off by at most 2^-25 of the largest one, n of them: n 2^-25 max |v|
  scores: products of fp16 values accumulated in fp32 (head_dim additions, one scaling), which move a weight by
      2 (head_dim + 2) 2^-24 sum |q k| / sqrt(head_dim), relative
  sums of weights and of weighted values in fp32, in any order: n 2^-24, relative to sum w |v| (twice: numerator, denominator)
Queries and the new key are compared from the oracle's fp16 rotation, whose bits the kernels reproduce."""
import numpy as np
import pytest

from oracle import pyoracle as orc
from tests import helpers as H

pytestmark = pytest.mark.gpu

NAN = 0x7e00
U32 = 2.0 ** -24
SHAPES = [(32, 8, 128), (8, 1, 128), (4, 4, 128), (16, 4, 64), (3, 3, 64), (8, 2, 32), (2, 2, 32)]


def say(*a):
    print(*a, flush=True)


def case(seed, B, prefix, tails, heads, tails_only, prefix_slack=0, own_slack=0, scale=1.0):
    """Random inputs; every cache row that holds no position the step may read is NaN."""
    Hq, Hkv, hd = heads
    rng = np.random.default_rng(seed)
    r64 = lambda n: (n + 63) // 64 * 64  # noqa: E731
    row0 = prefix if tails_only else 0
    positions = [prefix + t for t in tails]
    max_pos = r64(max(positions) + 1 - row0 + own_slack)
    pmax = r64(prefix + prefix_slack)
    kp, vp = np.full((Hkv, pmax, hd), NAN, np.uint16), np.full((Hkv, hd, pmax), NAN, np.uint16)
    kp[:, :prefix], vp[:, :, :prefix] = H.bits(rng.standard_normal((Hkv, prefix, hd))), H.bits(rng.standard_normal((Hkv, hd, prefix)))
    kcs, vcs = np.full((B, Hkv, max_pos, hd), NAN, np.uint16), np.full((B, Hkv, hd, max_pos), NAN, np.uint16)
    for z, t in enumerate(tails):
        a = prefix - row0
        kcs[z, :, a:a + t] = H.bits(rng.standard_normal((Hkv, t, hd)))
        vcs[z, :, :, a:a + t] = H.bits(rng.standard_normal((Hkv, hd, t)))
    qkv = H.bits(rng.standard_normal((B, (Hq + 2 * Hkv) * hd)) * scale)
    return dict(qkv=qkv, kp=kp, vp=vp, kcs=kcs, vcs=vcs, positions=positions, row0=row0, prefix=prefix, heads=heads)


def expected(c):
    """(out float64 [B, Hq*hd], tolerance of each element, K caches, V caches) after the step."""
    Hq, Hkv, hd = c["heads"]
    G, P, row0 = Hq // Hkv, c["prefix"], c["row0"]
    B = len(c["positions"])
    out, tol = np.zeros((B, Hq * hd)), np.zeros((B, Hq * hd))
    kcs, vcs = c["kcs"].copy(), c["vcs"].copy()
    for z, pos in enumerate(c["positions"]):
        line = c["qkv"][z:z + 1]
        q = H.f16(orc.rope(np.ascontiguousarray(line[:, :Hq * hd]), Hq, hd, pos)).reshape(Hq, hd)
        kn = orc.rope(np.ascontiguousarray(line[:, Hq * hd:(Hq + Hkv) * hd]), Hkv, hd, pos).reshape(Hkv, hd)
        kcs[z, :, pos - row0] = kn
        vcs[z, :, :, pos - row0] = line[0, (Hq + Hkv) * hd:].reshape(Hkv, hd)
        for h in range(Hkv):
            K = np.concatenate([H.f16(c["kp"][h, :P]), H.f16(kcs[z, h, P - row0:pos - row0 + 1])])
            V = np.concatenate([H.f16(c["vp"][h, :, :P]).reshape(hd, P), H.f16(vcs[z, h, :, P - row0:pos - row0 + 1])], 1)
            n = pos + 1
            for g in range(h * G, (h + 1) * G):
                s = K @ q[g] / np.sqrt(hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                o, spread = V @ w, np.abs(V) @ w
                size = (np.abs(K) @ np.abs(q[g])).max() / np.sqrt(hd)
                rel = 2.0 ** -11 + 2 * (hd + 2) * 2.0 ** -24 * size + 2 * n * 2.0 ** -24
                out[z, g * hd:(g + 1) * hd] = o
                tol[z, g * hd:(g + 1) * hd] = 2.0 ** -11 * np.abs(o) + rel * spread + n * 2.0 ** -25 * np.abs(V).max() * w.max()
    return out, tol, kcs, vcs


def run(gpu, c, **kw):
    return gpu.ops.attn_decode_rope_shared(c["qkv"], c["kp"] if c["prefix"] else None, c["vp"], c["prefix"], c["kcs"], c["vcs"],
                                           c["positions"], c["row0"], *c["heads"], **kw)


def verify(got, want):
    out, kcs, vcs = got
    w_out, tol, w_k, w_v = want
    err = np.abs(H.f16(out)[:, :w_out.shape[1]] - w_out)
    say("  worst error / tolerance: %.3f" % float(np.max(err / tol)))
    assert np.all(err <= tol)  # a NaN fails too
    assert np.array_equal(kcs, w_k) and np.array_equal(vcs, w_v)  # the new rows, and nothing else


@pytest.mark.parametrize("heads", SHAPES)
@pytest.mark.parametrize("tails_only", [False, True])
def test_every_head_shape(gpu, heads, tails_only):
    c = case(1, 3, 200, [0, 17, 70], heads, tails_only)
    say("shared attention", heads, "tails only" if tails_only else "full caches")
    verify(run(gpu, c), expected(c))


@pytest.mark.parametrize("prefix", [0, 1, 7, 8, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1025])
def test_prefix_lengths(gpu, prefix):
    c = case(2, 2, prefix, [0, 3], (8, 2, 128), True)
    say("prefix", prefix)
    verify(run(gpu, c), expected(c))


@pytest.mark.parametrize("tails", [[0], [1], [5, 0], [63, 64], [65, 1, 128], [300, 0, 2, 511]])
@pytest.mark.parametrize("prefix", [64, 77])
def test_tail_lengths(gpu, prefix, tails):
    """Tails that begin inside a tile (77 own rows are not read), at a tile, and sequences without one."""
    for tails_only in (False, True):
        c = case(3, len(tails), prefix, tails, (8, 2, 128), tails_only)
        say("tails", tails, "prefix", prefix, tails_only)
        verify(run(gpu, c), expected(c))


@pytest.mark.parametrize("B", [1, 2, 7, 8, 9, 16])
@pytest.mark.parametrize("heads", [(8, 2, 128), (16, 2, 128), (4, 1, 32), (2, 2, 64)])
def test_batches(gpu, B, heads):
    c = case(4, B, 150, [(5 * z) % 40 for z in range(B)], heads, False)
    say("batch", B, heads)
    verify(run(gpu, c), expected(c))


# The kernels have a one-launch form for short lengths and a two-launch form for long ones; a descriptor call is sized by its
# bounds, so that generous ones take the long form at any length.
def run_long(gpu, c):
    return gpu.ops.attn_decode_rope_shared(c["qkv"], c["kp"], c["vp"], c["prefix"], c["kcs"], c["vcs"], c["positions"], c["row0"],
                                           *c["heads"], dev=True, max_prefix=c["kp"].shape[1], max_tail=c["kcs"].shape[2] - 1)


@pytest.mark.parametrize("heads", SHAPES)
@pytest.mark.parametrize("tails_only", [False, True])
def test_every_head_shape_at_length(gpu, heads, tails_only):
    c = case(21, 4, 1400, [0, 17, 70, 129], heads, tails_only)
    say("shared attention, long", heads, "tails only" if tails_only else "full caches")
    verify(run(gpu, c), expected(c))


@pytest.mark.parametrize("prefix", [0, 1, 7, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (8, 2, 32)])
def test_short_lengths_in_the_long_form(gpu, prefix, heads):
    c = case(22, 3, prefix, [0, 5, 66], heads, True, prefix_slack=8192)
    say("long form, prefix", prefix, heads)
    verify(run_long(gpu, c), expected(c))


@pytest.mark.parametrize("prefix", [959, 960, 961, 1023, 1024, 1025, 1087, 2049])
@pytest.mark.parametrize("tails", [[0, 0], [1, 64], [63, 65], [200, 3]])
def test_long_prefix_edges(gpu, prefix, tails):
    c = case(23, 2, prefix, tails, (8, 2, 128), prefix % 2 == 0)
    say("prefix", prefix, "tails", tails)
    verify(run(gpu, c), expected(c))


@pytest.mark.parametrize("B", [1, 2, 4, 7, 8, 9, 16])
@pytest.mark.parametrize("heads", [(8, 2, 128), (16, 2, 128), (8, 2, 32), (2, 2, 64)])
def test_batches_at_length(gpu, B, heads):
    """One, two and four query tiles, batches that do not fill them."""
    c = case(24, B, 2100, [(11 * z) % 90 for z in range(B)], heads, True)
    say("batch, long", B, heads)
    verify(run(gpu, c), expected(c))


def test_tails_longer_than_the_prefix(gpu):
    c = case(25, 6, 65, [2000, 1, 700, 0, 1300, 64], (8, 2, 128), True)
    verify(run(gpu, c), expected(c))


def test_many_kv_heads(gpu):
    """More KV heads than one workgroup each fills the chip with."""
    c = case(26, 2, 300, [5, 40], (600, 600, 32), True, prefix_slack=8192)
    verify(run_long(gpu, c), expected(c))


def test_no_position_but_the_new_one(gpu):
    """Nothing cached at all: the output is the new value row."""
    c = case(5, 4, 0, [0, 0, 0, 0], (8, 2, 128), True)
    out, _, _ = run(gpu, c)
    Hq, Hkv, hd = c["heads"]
    v = c["qkv"][:, (Hq + Hkv) * hd:].reshape(4, Hkv, 1, hd)
    assert np.array_equal(out, np.broadcast_to(v, (4, Hkv, Hq // Hkv, hd)).reshape(4, Hq * hd))


def test_long_prefix_and_long_tails(gpu):
    c = case(6, 5, 5003, [0, 77, 1200, 64, 9], (8, 2, 128), True)
    verify(run(gpu, c), expected(c))


def test_scores_of_wide_range(gpu):
    """Scores in the hundreds: nearly all weight on a few positions, the running maximum moves often."""
    c = case(7, 3, 700, [40, 0, 130], (8, 2, 128), False, scale=30.0)
    verify(run(gpu, c), expected(c))


def test_strides_and_slack(gpu):
    """Projection and output rows with columns behind them, caches longer than what they hold."""
    Hq, Hkv, hd = 8, 2, 64
    c = case(8, 3, 100, [4, 0, 31], (Hq, Hkv, hd), False, prefix_slack=200, own_slack=300)
    want = expected(c)
    wide = np.full((3, c["qkv"].shape[1] + 24), NAN, np.uint16)
    wide[:, :c["qkv"].shape[1]] = c["qkv"]
    c["qkv"] = wide
    got = run(gpu, c, ldo=Hq * hd + 5)
    verify(got, want)
    assert np.all(got[0][:, Hq * hd:] == NAN)  # columns behind a row's result


def test_prefix_inside_one_of_the_caches(gpu):
    """The prefix read from sequence 1's own cache (row 0 = position 0), as forked caches have it."""
    c = case(9, 3, 90, [3, 20, 0], (8, 2, 128), False)
    want = expected(c)
    c["kcs"][1, :, :90], c["vcs"][1, :, :, :90] = c["kp"][:, :90], c["vp"][:, :, :90]
    out, kcs, vcs = gpu.ops.attn_decode_rope_shared(c["qkv"], 1, None, 90, c["kcs"], c["vcs"], c["positions"], 0, *c["heads"])
    want[2][1, :, :90], want[3][1, :, :, :90] = c["kp"][:, :90], c["vp"][:, :, :90]
    verify((out, kcs, vcs), want)


def test_descriptor_form_gives_the_same_result(gpu):
    for tails_only in (False, True):
        c = case(10, 5, 333, [0, 1, 50, 200, 7], (8, 2, 128), tails_only)
        host, dev = run(gpu, c), run(gpu, c, dev=True)
        assert all(np.array_equal(x, y) for x, y in zip(host, dev))  # same sizes, same order of sums
        want = expected(c)
        verify(dev, want)
        verify(run(gpu, c, dev=True, max_prefix=c["kp"].shape[1], max_tail=c["kcs"].shape[2] - 1 - (0 if tails_only else 333)), want)


def test_descriptor_beyond_its_bounds_is_clamped(gpu):
    """A descriptor that says more than the launch was sized for reads and writes inside the caches all the same: it is
    served as the clamped lengths."""
    c = case(11, 2, 128, [10, 30], (8, 2, 128), True)
    clamped = dict(c, positions=[128 + 10, 128 + 20])
    want = run(gpu, clamped, dev=True, max_tail=20)
    got = run(gpu, c, dev=True, max_tail=20)
    assert all(np.array_equal(x, y) for x, y in zip(got, want))
    wild = dict(c, positions=[128 + 10, 2 ** 31 - 1])
    got = run(gpu, wild, dev=True, max_tail=20)
    assert all(np.array_equal(x, y) for x, y in zip(got, want))
    got = run(gpu, dict(c, positions=[-5, 2 ** 31 - 1]), dev=True, max_tail=20)
    want = run(gpu, dict(c, positions=[128, 128 + 20]), dev=True, max_tail=20)
    assert all(np.array_equal(x, y) for x, y in zip(got, want))


def test_descriptor_with_a_prefix_beyond_the_own_caches_is_clamped(gpu):
    """Row 0 is position 0 and the prefix is longer than the caches: positions stay inside caches and (cos, sin) table."""
    c = dict(case(27, 2, 128, [0, 0], (8, 2, 128), True), row0=0)
    got = run(gpu, c, dev=True, max_prefix=128, max_tail=0)
    want = run(gpu, dict(c, prefix=63, positions=[63, 63]), dev=True, max_prefix=128, max_tail=0)
    assert all(np.array_equal(x, y) for x, y in zip(got, want))


def test_repeated_calls_give_equal_bits(gpu):
    c = case(12, 16, 1500, [(37 * z) % 200 for z in range(16)], (8, 2, 128), False)
    one, many = run(gpu, c), run(gpu, c, repeats=5)
    assert all(np.array_equal(x, y) for x, y in zip(one, many))


def test_captured_step_follows_the_descriptor(gpu):
    """A captured launch replayed while the descriptor's positions advance equals eager calls at every step."""
    import ctypes as C
    L, check, ops = gpu.lib(), gpu.capi.check, gpu.ops
    Hq, Hkv, hd = 8, 2, 128
    B, prefix, max_tail = 3, 130, 40
    c = case(13, B, prefix, [30, 2, 11], (Hq, Hkv, hd), True, own_slack=10)
    max_pos = c["kcs"].shape[2]
    Dev = gpu.capi.DevBuf
    d_q, d_kp, d_vp = Dev.from_host(c["qkv"]), Dev.from_host(c["kp"]), Dev.from_host(c["vp"])
    d_ks, d_vs = [Dev.from_host(k) for k in c["kcs"]], [Dev.from_host(v) for v in c["vcs"]]
    d_t = Dev.from_host(ops.rope_table(prefix + max_pos, hd))
    d_o, d_ws = Dev((B, Hq * hd), np.uint16), ops._zeroed(L.llm_attn_shared_workspace_bytes(Hq, Hkv, hd, B))

    def desc(positions):
        return np.frombuffer(bytes(ops.SharedDesc(d_kp.ptr, d_vp.ptr, prefix, prefix, (C.c_void_p * 16)(*[b.ptr for b in d_ks]),
                                                  (C.c_void_p * 16)(*[b.ptr for b in d_vs]), (C.c_int32 * 16)(*positions))), np.uint8)

    d_desc = Dev.from_host(desc(c["positions"]))
    stream, graph = C.c_void_p(), C.c_void_p()
    check(L.llm_stream_create(C.byref(stream)))
    check(L.llm_graph_capture_begin(stream))
    check(L.llm_attn_decode_rope_shared_dev(d_q.ptr, c["qkv"].shape[1], d_desc.ptr, 0, 0, 192, 192, max_tail, B, d_o.ptr, Hq * hd,
                                            d_t.ptr, Hq, Hkv, hd, max_pos, d_ws.ptr, stream))
    check(L.llm_graph_capture_end(stream, C.byref(graph)))
    state = dict(c)
    for step in range(5):
        positions = [p + step for p in c["positions"]]
        state["positions"] = positions
        d_desc.upload(desc(positions))
        d_o.zero()
        check(L.llm_graph_launch(graph, stream))
        check(L.llm_stream_sync(stream))
        got = d_o.download(), np.stack([b.download() for b in d_ks]), np.stack([b.download() for b in d_vs])
        say("replay", step)
        want = expected(state)
        verify(got, want)
        eager = run(gpu, state)  # eager work of other addresses between the replays
        assert np.all(np.abs(H.f16(eager[0]) - want[0]) <= want[1])
        state["kcs"], state["vcs"] = got[1], got[2]
    check(L.llm_graph_destroy(graph))
    check(L.llm_stream_destroy(stream))


def closely(c):
    """expected() with the tolerance of weights that enter the second product as the sum of two fp16 values.  Per element, with
    u = 2^-24, n the positions, size the largest sum |q k| / sqrt(head_dim), which bounds every score:
      half an fp16 step of the result, 2^-11 |o| + 2^-25
      the second product's weights: the first part rounded to 11 bits, the rest (2^-11 of the weight at most) too: 2^-22, relative,
        and 2^-25 of a scale on which the largest weight is 2^7 or more: n 2^-32 max |v|
      exp2: two units of the last place, 4 u; its argument: accumulation and scaling of the score (head_dim + 2) size u, three
        roundings of the factor 3 size u, one of the difference to the reference, whose value is below 2 size log2 e + 16, and
        two more of that kind where references are joined: 3 (2 size + 12) u
      sums of weights and of weighted values, in any order: n u
    all but the first two of them once in the numerator and once in the denominator."""
    out, _, kcs, vcs = expected(c)
    Hq, Hkv, hd = c["heads"]
    G, P, row0 = Hq // Hkv, c["prefix"], c["row0"]
    tol, u = np.zeros_like(out), 2.0 ** -24
    for z, pos in enumerate(c["positions"]):
        q = H.f16(orc.rope(np.ascontiguousarray(c["qkv"][z:z + 1, :Hq * hd]), Hq, hd, pos)).reshape(Hq, hd)
        for h in range(Hkv):
            K = np.concatenate([H.f16(c["kp"][h, :P]), H.f16(kcs[z, h, P - row0:pos - row0 + 1])])
            V = np.abs(np.concatenate([H.f16(c["vp"][h, :, :P]).reshape(hd, P), H.f16(vcs[z, h, :, P - row0:pos - row0 + 1])], 1))
            n = pos + 1
            for g in range(h * G, (h + 1) * G):
                s = K @ q[g] / np.sqrt(hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                size = (np.abs(K) @ np.abs(q[g])).max() / np.sqrt(hd)
                rel = 2.0 ** -22 + 2 * u * (4 + (hd + 2) * size + 3 * size + 3 * (2 * size + 12) + n)
                at = slice(g * hd, (g + 1) * hd)
                tol[z, at] = 2.0 ** -11 * np.abs(out[z, at]) + 2.0 ** -25 + rel * (V @ w) + n * 2.0 ** -32 * V.max() * w.max()
    return out, tol, kcs, vcs


@pytest.mark.parametrize("heads", SHAPES)
@pytest.mark.parametrize("prefix", [90, 1500])
def test_weights_are_held_in_more_than_the_operands_type(gpu, heads, prefix):
    """Few positions of like weight and values of either sign: a weight in a single fp16 shows beside the result's rounding."""
    c = case(31, 4, prefix, [0, 17, 70, 33], heads, False, scale=1.5)
    say("weights", heads, prefix)
    verify(run(gpu, c), closely(c))


@pytest.mark.parametrize("gap", [6, 10, 14, 18, 22, 25, 28, 31])
@pytest.mark.parametrize("n", [120, 6000])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 64), (2, 2, 32)])
def test_many_small_weights_count(gpu, heads, n, gap):
    """One position far ahead of n others, each 2^-gap of its weight: together they are a part of the result at any gap."""
    Hq, Hkv, hd = heads
    c = case(32, 2, n, [0, 3], heads, False)
    q = np.tile(np.random.default_rng(gap).standard_normal(hd), Hq)
    for z in range(2):
        c["qkv"][z, :Hq * hd] = H.bits(q)
        c["qkv"][z, Hq * hd:(Hq + Hkv) * hd] = 0                    # the new key: score 0
        c["qkv"][z, (Hq + Hkv) * hd:] = H.bits(1.0)
    turned = H.f16(orc.rope(np.ascontiguousarray(c["qkv"][:1, :Hq * hd]), Hq, hd, n)).reshape(Hq, hd)[0]
    c["kp"][:, :n], c["vp"][:, :, :n] = 0, H.bits(1.0)
    c["kcs"][1, :, n:n + 3], c["vcs"][1, :, :, n:n + 3] = 0, H.bits(1.0)
    ahead = n // 3
    c["kp"][:, ahead] = H.bits(turned * (gap * np.log(2.0) * np.sqrt(hd) / (turned @ turned)))
    c["vp"][:, :, ahead] = 0
    say("gap", gap, "of", n, heads)
    verify(run(gpu, c), closely(c))


@pytest.mark.parametrize("heads", [(8, 2, 128), (8, 1, 128), (4, 4, 64), (8, 2, 32)])
@pytest.mark.parametrize("prefix", [100, 3000])
@pytest.mark.parametrize("scale", [300.0, 12000.0])
def test_scores_of_any_magnitude(gpu, heads, prefix, scale):
    """Queries and keys far up in their type's range (scores to 10^9 and more): the best position takes all the weight wherever it is
    ahead by more than a score's error, (head_dim + 2) 2^-24 times the sum of |q k| (twice, for the two scores), and 40 (e^-40 of n
    values of like size is far below half a step)."""
    Hq, Hkv, hd = heads
    c = case(33, 2, prefix, [0, 40], heads, False)
    for name in ("qkv", "kp", "kcs"):
        x = H.f16(c[name]) * scale
        if name == "qkv":
            x[:, (Hq + Hkv) * hd:] /= scale
        c[name] = np.where(np.isnan(x), np.uint16(NAN), H.bits(np.clip(np.nan_to_num(x), -40000.0, 40000.0)))
    got, kcs, vcs = run(gpu, c)
    _, _, w_k, w_v = expected(c)
    assert np.array_equal(kcs, w_k) and np.array_equal(vcs, w_v)
    assert np.all(np.isfinite(H.f16(got)))
    seen = 0
    for z, pos in enumerate(c["positions"]):
        q = H.f16(orc.rope(np.ascontiguousarray(c["qkv"][z:z + 1, :Hq * hd]), Hq, hd, pos)).reshape(Hq, hd)
        for g in range(Hq):
            h = g // (Hq // Hkv)
            K = np.concatenate([H.f16(c["kp"][h, :prefix]), H.f16(w_k[z, h, prefix:pos + 1])])
            V = np.concatenate([c["vp"][h, :, :prefix], w_v[z, h, :, prefix:pos + 1]], 1)
            s, off = K @ q[g] / np.sqrt(hd), 2 * (hd + 2) * U32 * (np.abs(K) @ np.abs(q[g])).max() / np.sqrt(hd)
            order = np.argsort(s)
            if s[order[-1]] - s[order[-2]] > off + 40:
                seen += 1
                assert np.array_equal(got[z, g * hd:(g + 1) * hd], V[:, order[-1]]), (z, g)
    say("rows with one position ahead:", seen, "of", 2 * Hq)
    assert seen >= Hq


@pytest.mark.parametrize("fill", [0x00, 0xff, 0x7f])
def test_a_workspace_of_any_contents(gpu, monkeypatch, fill):
    """Zeros, NaN or large numbers in the workspace: a call reads nothing there that it did not write, in any of its forms."""
    def filled(nbytes):
        return gpu.capi.DevBuf.from_host(np.full(nbytes + 3 & ~3, fill, np.uint8))

    for prefix, tails, heads in ((1400, [0, 17, 70, 129], (8, 2, 128)), (65, [2000, 1, 700], (8, 2, 128)), (3000, [0, 0], (4, 4, 64)),
                                 (200, [3, 9], (8, 2, 32))):
        c = case(34, len(tails), prefix, tails, heads, True)
        with monkeypatch.context() as m:
            zeroed = run(gpu, c)
            m.setattr(gpu.ops, "_zeroed", filled)
            assert all(np.array_equal(x, y) for x, y in zip(run(gpu, c), zeroed))
            want = expected(c)
            verify(run(gpu, c, dev=True, max_prefix=c["kp"].shape[1], max_tail=c["kcs"].shape[2] - 1), want)


@pytest.mark.parametrize("prefix,row0", [(200, 1), (200, 7), (200, 64), (200, 199), (1400, 8), (1400, 199), (1400, 1300)])
def test_own_caches_that_begin_inside_the_prefix(gpu, prefix, row0):
    """Row 0 of the own caches is a position of the prefix: their rows in front of the prefix's end are not read."""
    lead = prefix - row0
    c = case(35, 3, prefix, [0, 17, 130], (8, 2, 128), True, own_slack=lead)
    kcs, vcs = np.full_like(c["kcs"], NAN), np.full_like(c["vcs"], NAN)
    kcs[:, :, lead:lead + 130], vcs[:, :, :, lead:lead + 130] = c["kcs"][:, :, :130], c["vcs"][:, :, :, :130]
    c.update(kcs=kcs, vcs=vcs, row0=row0)
    say("prefix", prefix, "row 0 at", row0)
    want = closely(c)
    verify(run(gpu, c), want)
    verify(run(gpu, c, dev=True, max_prefix=c["kp"].shape[1], max_tail=kcs.shape[2] - 1), want)
