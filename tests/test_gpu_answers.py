"""Several answers to one prompt through the engine: forked caches, batched steps that read the shared prompt once, log
probabilities -- against caches that were filled on their own, the same steps without sharing, and 64-bit log probabilities of
the engine's own logits."""
import os
import subprocess

import numpy as np
import pytest

from tests import helpers as H

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module")
def tiny(gpu):
    cfg = gpu.engine.config("tiny", max_pos=1024)
    model = gpu.engine.Model.seeded(cfg, 77).to_device()
    yield gpu, cfg, model
    model.close()


def engines(gpu, cfg, model, n, **kw):
    return [gpu.engine.Engine(model, cfg, **kw) for _ in range(n)]


def close_all(es):
    for e in es:
        e.close()


def log_softmax(bits, t=1.0):
    x = H.f16(bits) / np.float64(np.float32(t))
    x = x - x.max()
    return x - np.log(np.exp(x).sum())


def walk(gpu, es, prompt, steps, tokens, fill):
    """Fills the engines with the prompt (fill(es)) and takes the given steps; returns the logits after each."""
    fill(es)
    seen = []
    for s in range(steps):
        gpu.engine.Engine.decode_batch(es, tokens[s][:len(es)])
        seen.append([es[0].batch_logits(b) for b in range(len(es))])
    return seen


@pytest.mark.parametrize("batch,n_prompt", [(2, 1), (3, 77), (8, 520), (16, 300)])
@pytest.mark.parametrize("use_graph", [True, False])
def test_forks_step_like_caches_filled_on_their_own(tiny, batch, n_prompt, use_graph):
    """Every row of every step within the model's tolerance of the batched step that shares nothing, and of a shared step of
    forks against the same forks without sharing."""
    gpu, cfg, model = tiny
    rng = np.random.default_rng(batch)
    prompt = gpu.engine.seeded_tokens(5, n_prompt, cfg.vocab)
    tokens = rng.integers(0, cfg.vocab, size=(6, batch))
    say("forks", batch, "prompt", n_prompt, "graph", use_graph)

    def own(es):
        for e in es:
            e.prefill(prompt)

    def forked(es):
        es[0].prefill(prompt)
        es[0].fork(es[1:])

    a = engines(gpu, cfg, model, batch, use_graph=use_graph)
    want = walk(gpu, a, prompt, 6, tokens, own)
    assert a[0].shared_prefix_steps() == 0
    close_all(a)
    got = {}
    for mode in (0, 1, 2):
        b = engines(gpu, cfg, model, batch, use_graph=use_graph)
        b[0].set_shared_prefix(mode)
        got[mode] = walk(gpu, b, prompt, 6, tokens, forked)
        shared = b[0].shared_prefix_steps()
        assert shared == (0 if mode == 0 else 6 if mode == 2 else 6 if n_prompt >= 512 and batch * n_prompt >= 4096 else 0)
        assert all(e.pos == n_prompt + 6 for e in b)
        close_all(b)
    for s in range(6):
        for z in range(batch):
            # a forked cache holds the same rows: without sharing, the same bits as caches filled on their own
            assert np.array_equal(got[0][s][z], want[s][z]), (s, z)
            for mode in (1, 2):
                assert H.mixed_err(got[mode][s][z], want[s][z]) <= H.TOL, (mode, s, z)


def test_branches_of_branches(tiny):
    """Beams: a cache branches again and again, destinations that share rows with it take only the rest; every cache equals one
    that went the same way alone."""
    gpu, cfg, model = tiny
    es = engines(gpu, cfg, model, 4)
    way = [[int(t) for t in gpu.engine.seeded_tokens(9, 40, cfg.vocab)]] * 4
    es[0].set_shared_prefix(2)
    es[0].prefill(way[0])
    es[0].fork(es[1:])
    rng = np.random.default_rng(1)
    for r in range(14):  # more generations than a cache remembers marks
        tok = [int(t) for t in rng.integers(0, cfg.vocab, 4)]
        gpu.engine.Engine.decode_batch(es, tok)
        way = [w + [t] for w, t in zip(way, tok)]
        src, dst = r % 4, (r + 1 + r // 4 % 3) % 4
        if src != dst:
            es[src].fork([es[dst]])
            way[dst] = list(way[src])
    tok = [int(t) for t in rng.integers(0, cfg.vocab, 4)]
    gpu.engine.Engine.decode_batch(es, tok)
    assert es[0].shared_prefix_steps() == 15
    alone = gpu.engine.Engine(model, cfg)
    for z in range(4):
        alone.reset()
        alone.prefill(way[z])
        alone.decode(tok[z])
        err = H.mixed_err(es[0].batch_logits(z), alone.logits())
        say("branch", z, "error", err)
        assert err <= H.TOL
    alone.close()
    close_all(es)


def test_a_fork_takes_every_call(tiny):
    """Single steps, prompt passes, generation and inference() on a fork equal those on the source, and neither changes the other."""
    gpu, cfg, model = tiny
    a, b = engines(gpu, cfg, model, 2)
    prompt = [int(t) for t in gpu.engine.seeded_tokens(3, 50, cfg.vocab)]
    b.prefill([1, 2, 3])  # what a destination held before is gone
    first, _ = a.prefill(prompt)
    a.fork([b])
    assert b.pos == 50 and np.array_equal(a.logits(), b.logits())
    for t in (first, 17, 4000):
        ta, tb = a.decode(t)[0], b.decode(t)[0]
        assert ta == tb and np.array_equal(a.logits(), b.logits())
    c = gpu.engine.Engine(model, cfg)
    a.fork([c])
    more = [int(t) for t in gpu.engine.seeded_tokens(4, 20, cfg.vocab)]
    assert a.prefill(more)[0] == c.prefill(more)[0] and np.array_equal(a.logits(), c.logits())
    a.fork([c])
    ga, _ = a.generate([5], 8)
    gc, _ = c.generate([5], 8)
    assert np.array_equal(ga, gc)
    # the fork continues a token list through inference() without computing its rows again
    b.reset()
    assert b.pos == 0
    b.prefill(prompt)
    b.fork([c])
    assert b.inference(prompt + [7]) == c.inference(prompt + [7]) and c.pos == 51
    # a reset cache shares nothing any more
    b.set_shared_prefix(2)
    b.reset()
    b.prefill(prompt + [7])
    gpu.engine.Engine.decode_batch([b, c], [1, 2])
    assert b.shared_prefix_steps() == 0
    close_all([a, b, c])


def test_fork_of_an_empty_cache(tiny):
    gpu, cfg, model = tiny
    a, b = engines(gpu, cfg, model, 2)
    b.prefill([4, 5])
    a.fork([b])
    assert b.pos == 0
    assert a.prefill([9, 8, 7])[0] == b.prefill([9, 8, 7])[0] and np.array_equal(a.logits(), b.logits())
    close_all([a, b])


def check_logprobs(bits, t, ids, k, got):
    """got: (logprob, entropy, top ids, top logprob) of one row, against 64 bits.  Tolerance: 2^-24 times the additions that follow
    one another (a lane sees every 256th logit at most, 64 joins), 12 roundings of terms no larger than |log p| + 1, and as much
    again for the sums' terms, whose weighted mean is below 2 log(vocab)."""
    lp, ent, ti, tl = got
    want = log_softmax(bits, t)
    unit = 2.0 ** -24
    tol = lambda x: unit * (len(want) / 256 + 64 + 12 * (np.abs(x) + 1) + 24 * np.log(len(want)))  # noqa: E731
    assert np.all(np.abs(lp - want[ids]) <= tol(want[ids]))
    h = -(np.exp(want) * want).sum()
    assert abs(ent - h) <= (h + 2) * unit * (len(want) / 256 + 64 + 24 * np.log(len(want)))
    order = np.lexsort((np.arange(len(want)), -(H.f16(bits) + 0.0)))[:k]
    assert np.array_equal(ti, order) and np.all(np.abs(tl - want[order]) <= tol(want[order]))


def test_log_probabilities_of_steps(tiny):
    gpu, cfg, model = tiny
    es = engines(gpu, cfg, model, 5)
    es[0].prefill([int(t) for t in gpu.engine.seeded_tokens(3, 30, cfg.vocab)])
    check_logprobs(es[0].logits(), 0.7, [5, 4095, 5], 20, es[0].logprobs([5, 4095, 5], 20, 0.7))
    assert np.isnan(es[0].logprobs([4096])[0][0]) and np.isnan(es[0].logprobs([-1])[0][0])
    es[0].fork(es[1:])
    ids = np.array([[1, 2], [3, 4], [5, 6], [7, 8], [4095, 0]])
    nxt = gpu.engine.Engine.decode_batch(es, [10, 11, 12, 13, 14])
    for t in (1.0, 1.3):
        lp, ent, ti, tl = es[0].batch_logprobs(ids, 3, t)
        for z in range(5):
            check_logprobs(es[0].batch_logits(z), t, ids[z], 3, (lp[z], ent[z], ti[z], tl[z]))
            assert ti[z][0] == nxt[z]  # the likeliest alternative is the greedy id
    lp, ent, _, _ = es[0].batch_logprobs([7, 7, 7, 7, 7])
    assert lp.shape == (5, 1) and np.all(ent > 0)
    # a smaller batch behind a larger one: its rows only
    gpu.engine.Engine.decode_batch(es[:2], [1, 2])
    lp, ent, ti, tl = es[0].batch_logprobs([[5], [6]], 1)
    for z in range(2):
        check_logprobs(es[0].batch_logits(z), 1.0, [5 + z], 1, (lp[z], ent[z], ti[z], tl[z]))
    close_all(es)


@pytest.mark.parametrize("n", [1, 2, 33, 700])
def test_score_of_a_text(tiny, n):
    """Every row of a scored pass against single steps over the same text, and the cache it leaves against a prompt pass."""
    gpu, cfg, model = tiny
    text = [int(t) for t in gpu.engine.seeded_tokens(n, n, cfg.vocab)]
    a, b = engines(gpu, cfg, model, 2)
    a.prefill([3, 1, 4])
    b.prefill([3, 1, 4])
    nxt, lp, ent, ti, tl = a.score(text, k=4)
    say("score", n)
    assert a.pos == 3 + n and np.isnan(lp[-1]) and not np.any(np.isnan(lp[:-1]))
    want, _ = b.prefill(text)
    assert nxt == want and np.array_equal(a.logits(), b.logits())  # the pass itself is a prompt pass
    assert a.decode(9)[0] == b.decode(9)[0] and np.array_equal(a.logits(), b.logits())
    b.reset()
    b.prefill([3, 1, 4])
    rows = range(n) if n < 40 else range(0, 40)
    for i in rows:
        b.decode(text[i])
        logits = log_softmax(b.logits())
        # logits within the model's tolerance (single steps and a pass round differently): log probabilities within twice that
        bound = 2 * H.TOL * (1 + np.abs(H.f16(b.logits())).max())
        if i + 1 < n:
            assert abs(lp[i] - logits[text[i + 1]]) <= bound
        assert np.all(np.abs(tl[i] - logits[ti[i]]) <= bound)
        assert np.all(np.diff(tl[i]) <= 0)
        assert abs(ent[i] + (np.exp(logits) * logits).sum()) <= bound * (2 + np.log(cfg.vocab))
    close_all([a, b])


def test_answers_command(gpu):
    """llama3_main --answers: sampled side by side, listed by their log probability."""
    exe = os.path.join(os.path.dirname(gpu.LIB_PATH), "llama3_main")
    p = subprocess.run([exe, "--config", "tiny", "--prompt-len", "600", "--decode", "5", "--answers", "8"], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stdout + p.stderr
    lines = [l for l in p.stdout.splitlines() if l.startswith("answer ")]
    means = [float(l.split("probability ")[1].split(":")[0]) for l in lines]
    assert len(lines) == 8 and means == sorted(means, reverse=True) and all(len(l.split(":")[1].split()) == 5 for l in lines)
    assert "batched steps that read the prompt's rows once: 4 of 4" in p.stdout


BATCHED = "a.prefill([1]); b.prefill([2]); E = pkg.engine.Engine; E.decode_batch([a, b], [3, 4]); "


def test_log_probabilities_behind_a_batched_step(tiny):
    """A step of a cache's own behind a batched one makes the last row its own again, in a fork of it too."""
    gpu, cfg, model = tiny
    a, b = engines(gpu, cfg, model, 2)
    a.prefill([5, 6, 7])
    a.fork([b])
    gpu.engine.Engine.decode_batch([a, b], [8, 9])
    a.decode(10)
    a.fork([b])
    ids = [1, 2, 3]
    of_a, of_b = a.logprobs(ids, 5), b.logprobs(ids, 5)
    assert all(np.array_equal(p, q) for p, q in zip(of_a, of_b))
    check_logprobs(a.logits(), 1.0, ids, 5, of_a)
    close_all([a, b])


@pytest.mark.parametrize("code", ["a.logprobs([1])", "b.logprobs([1])", "c = E(m, cfg); b.fork([c]); c.logprobs([1])"])
def test_log_probabilities_of_a_batched_row_are_refused(gpu, code):
    test_refusals_end_with_a_message(gpu, BATCHED + code, "batched step")


REFUSALS = [
    ("a.fork([])", "destinations"), ("a.fork([a])", "is the source"), ("a.fork([b, b])", "share a cache"),
    ("a.fork([pkg.engine.Engine(m, pkg.engine.config('tiny', max_pos=128))])", "different configuration"),
    ("a.fork([b] * 17)", "destinations"), ("a.set_shared_prefix(3)", "mode"), ("a.logprobs([1])", "no row"),
    ("a.batch_logprobs([1])", "no batch step"), ("a.prefill([1]); a.logprobs([1] * 17)", "given tokens"), ("a.prefill([1]); a.logprobs([1], 33)", "alternatives"),
    ("a.prefill([1]); a.logprobs([1], 1, 0.0)", "temperature"), ("a.score([])", "at least one token"), ("a.score([1] * 2000)", "exceeds"), ("a.score([4096])", "vocabulary"),
]


@pytest.mark.parametrize("code,text", REFUSALS)
def test_refusals_end_with_a_message(gpu, code, text):
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", "import __graft_entry__ as ge; pkg = ge.load_package(); cfg = pkg.engine.config('tiny')\n"
                        "m = pkg.engine.Model.seeded(cfg, 1).to_device(); a, b = pkg.engine.Engine(m, cfg), pkg.engine.Engine(m, cfg)\n" + code],
                       cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=120)
    assert p.returncode == 1 and text in p.stdout, p.stdout + p.stderr


def test_batch_log_probabilities_take_one_row_per_sequence(tiny):
    """Ids of more or of fewer sequences than the last batched step had are refused in front of the library's call, which reads and
    writes as many rows as the step had; no ids at all are no given tokens."""
    gpu, cfg, model = tiny
    es = engines(gpu, cfg, model, 5)
    es[0].prefill([1, 2, 3])
    es[0].fork(es[1:])
    gpu.engine.Engine.decode_batch(es, [4, 5, 6, 7, 8])
    assert gpu.lib().llama3_batch_rows(es[0].cache) == 5 and gpu.lib().llama3_batch_rows(es[1].cache) == 0
    for ids in ([7], [[7]], [1, 2, 3, 4], [1, 2, 3, 4, 5, 6], [[1, 2]] * 16):
        with pytest.raises(ValueError, match="had 5"):
            es[0].batch_logprobs(ids, 2)
    for none in ([], [[], [], [], [], []]):
        lp, ent, ti, tl = es[0].batch_logprobs(none, 2)
        assert lp.shape == (5, 0) and ti.shape == (5, 2)
        for z in range(5):
            check_logprobs(es[0].batch_logits(z), 1.0, [], 2, (lp[z], ent[z], ti[z], tl[z]))
    assert es[0].batch_logprobs([1, 2, 3, 4, 5])[0].shape == (5, 1)
    gpu.engine.Engine.decode_batch(es[:2], [1, 2])
    with pytest.raises(ValueError, match="had 2"):
        es[0].batch_logprobs([1, 2, 3, 4, 5])
    close_all(es)


@pytest.mark.parametrize("over", ["rope_theta=10000.0", "rms_eps=1e-6"])
@pytest.mark.parametrize("call", ["a.fork([c])", "a.fork([b, c])", "E.decode_batch([a, c], [1, 2])", "E.decode_batch([c, b], [1, 2])"])
def test_caches_that_rotate_or_normalise_otherwise_are_refused(gpu, over, call):
    """Their rows, and the (cos, sin) table that a batched step takes from its first cache, would not fit together."""
    test_refusals_end_with_a_message(gpu, "E = pkg.engine.Engine; c = E(m, pkg.engine.config('tiny', %s)); a.prefill([1]); %s" % (over, call),
                                     "different configuration")


OTHER = "E = pkg.engine.Engine; n = pkg.engine.Model.seeded(cfg, 2).to_device(); c = E(n, cfg); a.prefill([1, 2]); a.fork([c]); "


@pytest.mark.parametrize("call", ["c.decode(3)", "c.prefill([3])", "c.generate([3], 2)", "c.score([3])", "E.decode_batch([c, b], [1, 2])",
                                  "E.decode_batch([a, c], [1, 2]); print('taken'); c.decode(3)", "c.fork([b]); b.fork([c]); c.decode(3)"])
def test_forked_rows_do_not_continue_under_another_model(gpu, call):
    """A fork into an engine of other weights holds rows that those did not compute; steps of the source's model take it."""
    test_refusals_end_with_a_message(gpu, OTHER + call, "another model")


def test_a_reset_fork_takes_any_model(tiny):
    gpu, cfg, model = tiny
    other = gpu.engine.Model.seeded(cfg, 5).to_device()
    a, b, c = engines(gpu, cfg, model, 1) + engines(gpu, cfg, other, 2)
    a.prefill([1, 2, 3])
    a.fork([b])
    b.reset()
    assert b.prefill([4, 5])[0] == c.prefill([4, 5])[0] and np.array_equal(b.logits(), c.logits())
    c.fork([a])
    a.reset()
    a.prefill([1, 2, 3])
    c.fork([b])
    assert b.decode(6)[0] == c.decode(6)[0]
    close_all([a, b, c])
    other.close()


def test_batch_log_probabilities_are_gone_with_a_reset(gpu):
    test_refusals_end_with_a_message(gpu, BATCHED + "print(a.batch_logprobs([1, 2])[0].shape); a.reset(); "
                                     "assert pkg.lib().llama3_batch_rows(a.cache) == 0; a.prefill([1]); a.batch_logprobs([1, 2])", "no batch step")


@pytest.mark.parametrize("n", [1, 2, 5, 33, 513, 514, 700])
def test_the_last_row_of_a_score_is_that_of_the_returned_id(tiny, n):
    gpu, cfg, model = tiny
    a = engines(gpu, cfg, model, 1)[0]
    for seed in range(4):
        a.reset()
        for t in (1.0, 0.4):
            nxt, lp, ent, ti, tl = a.score([int(x) for x in gpu.engine.seeded_tokens(seed + 1, n, cfg.vocab)], k=7, temperature=t)
            _, e, i, l = a.logprobs(k=7, temperature=t)
            assert ti[-1][0] == nxt and np.isnan(lp[-1])
            assert np.float32(e) == ent[-1] and np.array_equal(i, ti[-1]) and np.array_equal(l.view(np.uint32), tl[-1].view(np.uint32))
            if n > 511:
                a.reset()
    a.close()


@pytest.mark.parametrize("temperature", ["0.0", "-1.0", "float('nan')", "float('inf')"])
def test_a_refused_score_appends_nothing(gpu, temperature):
    """The temperature is looked at in front of the pass, like the other arguments."""
    test_refusals_end_with_a_message(gpu, "import ctypes; cb = ctypes.CFUNCTYPE(None, ctypes.c_char_p)(lambda s: print('refused at', a.pos, s, flush=True))\n"
                                     "pkg.lib().llama3_set_error_handler(cb); a.prefill([1]); a.score([2, 3], 1, %s)" % temperature, "refused at 1 ")
