"""The operators behind several scored answers to one prompt, as cases to be measured: decode attention of a batch whose
sequences share a prefix (llm_attn_decode_rope_shared), rows of a KV cache copied into other caches (llm_kv_fork), and log
probabilities of given tokens with entropy and top alternatives (llm_logprobs).

Every operator exists here twice: in its plain form, from elementary torch operations (`own` false), and as the call a
program makes of the library (`own` true).  Cache layouts are the library's: K [kv heads][max_pos][head_dim],
V [kv heads][head_dim][max_pos], fp16.
"""
import ctypes
import math

import torch

own = False

# (query heads, KV heads, head size): LLaMA3-8B, the tiny model, and the other head sizes and groups that are built
HEADS = [(32, 8, 128), (8, 2, 32), (16, 4, 64), (64, 8, 128), (8, 8, 64)]


def listed():
    return [
        # sixteen answers to an 8192-token prompt, 256 tokens into them; every cache holds the prompt too (forked caches)
        _attn("shared 16 x (8192 + 256)", 16, 8192, 256, HEADS[0], False),
        # the same with caches that hold the answers only, at a long prompt and answers of uneven lengths
        _attn("shared 16 x (32768 + 1024)", 16, 32768, 1024, HEADS[0], True),
        # two answers to a short prompt with the tiny model: the smallest call, where latency counts
        _attn("shared 2 x (300 + 5)", 2, 300, 5, HEADS[1], False),
        # an odd batch on groups of eight query heads, odd lengths
        _attn("shared 5 x (5003 + 77)", 5, 5003, 77, HEADS[3], True),
        # no sharing among heads, small heads, the first tokens behind a prompt
        _attn("shared 7 x (1023 + 1)", 7, 1023, 1, HEADS[4], False),
        # a decode step that reports its token's probability and the twenty best alternatives
        _logp("logprobs 1 x 128256 top 20", 1, 128256, 0, 20, 1, 1.0, False),
        # the same for a batched step, under the sampler's temperature
        _logp("logprobs 16 x 128256 top 5", 16, 128256, 0, 5, 1, 0.7, False),
        # a text is scored: the log probability of every next token, and the token that was the likeliest there
        _logp("logprobs 2048 x 128256 top 1", 2048, 128256, 0, 1, 1, 1.0, False),
        # a few candidates per row under a grammar's mask, odd vocabulary, rows that start anywhere
        _logp("logprobs 37 x 32003 masked", 37, 32003, 5, 10, 4, 1.0, True),
        # a prompt's cache becomes the caches of four answers (8B: 32 layers)
        _fork("fork 2048 rows to 4", 32, 8, 128, 2560, 0, 2560, 0, 2048, 4),
        # an answer of 1000 tokens joins the rows of its prompt: other row numbers, not aligned alike
        _fork("fork 1000 rows, moved", 32, 8, 128, 1024, 0, 4096, 1037, 1000, 1),
        # an answer branches after a few tokens: two short copies
        _fork("fork 33 rows to 2", 32, 8, 128, 2048, 1021, 2048, 1021, 33, 2),
    ]


def draw(rng):
    kind = rng.choice(["shared", "logprobs", "fork"])
    if kind == "shared":
        heads = rng.choice(HEADS)
        return _attn(None, rng.randint(1, 16), _spread(rng, 1, 32768 if heads[0] < 64 else 16384), _spread(rng, 1, 1024), heads,
                     rng.random() < 0.5)
    if kind == "logprobs":
        vocab = _spread(rng, 64, 131072)
        rows = _spread(rng, 1, min(2048, 2048 * 128256 // vocab))
        return _logp(None, rows, vocab, rng.choice([0, 0, rng.randint(1, 40)]), rng.choice([0, 1, 5, 20, rng.randint(1, 32)]),
                     rng.choice([0, 1, 1, rng.randint(1, 16)]) or 1, rng.choice([1.0, 0.7, rng.uniform(0.3, 2.0)]),
                     rng.random() < 0.3)
    heads = rng.choice(HEADS)
    layers, n, dsts = rng.randint(1, 32), _spread(rng, 1, 2048), rng.randint(1, 16)
    dsts = max(1, min(dsts, 32 * 2048 * 5 * 1024 // (layers * n * heads[1] * heads[2]) - 1))
    src_row = rng.randint(0, 512)
    dst_row = src_row if rng.random() < 0.5 else rng.randint(0, 512)
    return _fork(None, layers, heads[1], heads[2], _round64(src_row + n), src_row, _round64(dst_row + n), dst_row, n, dsts)


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _round64(n):
    return (n + 63) // 64 * 64


def _named(name, case):
    return dict(case, name=name) if name else case


def _attn(name, batch, prefix, tail, heads, tails_only):
    """tail: rows that the longest sequence has behind the prefix; the others have fewer (_tails)."""
    return _named(name, {"op": "shared", "batch": batch, "prefix": prefix, "tail": tail, "heads": heads[0], "kv_heads": heads[1],
                         "head_dim": heads[2], "tails_only": tails_only})


def _logp(name, rows, vocab, pad, k, n_ids, temperature, masked):
    """pad: elements between the end of a row and the next one."""
    return _named(name, {"op": "logprobs", "rows": rows, "vocab": vocab, "pad": pad, "k": k, "n_ids": n_ids,
                         "temperature": temperature, "masked": masked})


def _fork(name, layers, kv_heads, head_dim, src_max, src_row, dst_max, dst_row, n, dsts):
    return _named(name, {"op": "fork", "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "src_max": src_max,
                         "src_row": src_row, "dst_max": dst_max, "dst_row": dst_row, "n": n, "dsts": dsts})


def _tails(case):
    """Rows behind the prefix that each sequence of a case has cached: the last the most, the others a spread below it."""
    return [(case["tail"] * (2 * z + 3) // (2 * case["batch"] + 1)) for z in range(case["batch"])]


def work(case):
    if case["op"] == "shared":
        hq, hkv, hd, b = case["heads"], case["kv_heads"], case["head_dim"], case["batch"]
        tails = _tails(case)
        rows = case["prefix"] + sum(tails)
        moved = 4 * rows * hkv * hd + 2 * b * (hq + 2 * hkv) * hd + 4 * b * hkv * hd + 2 * b * hq * hd + 4 * b * hd
        return {"bytes": moved, "flops": 4 * hq * hd * sum(case["prefix"] + t + 1 for t in tails)}
    if case["op"] == "logprobs":
        rows = case["rows"]
        return {"bytes": 2 * rows * case["vocab"] + 4 * rows * (2 * case["n_ids"] + 1 + 2 * case["k"]),
                "flops": 6 * rows * case["vocab"]}
    one = 4 * case["n"] * case["layers"] * case["kv_heads"] * case["head_dim"]
    return {"bytes": one * (1 + case["dsts"]), "flops": 0}


def _randn(gen, *shape):
    """Normal fp16 values, made in parts of 2^26 so that a large cache needs no larger fp32 copy."""
    out = torch.empty(shape, dtype=torch.float16, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 26):
        part = flat[at:at + (1 << 26)]
        part.copy_(torch.randn(part.numel(), generator=gen, device="cuda"))
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    {"shared": _prepare_shared, "logprobs": _prepare_logprobs, "fork": _prepare_fork}[case["op"]](s, case, gen)
    if own:
        _prepare_call(s, case)
    return s


def _prepare_shared(s, case, gen):
    """Caches as prompt passes and earlier steps leave them, the projection row of every sequence's new token, and the
    (cos, sin) table."""
    b, hq, hkv, hd, prefix = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["prefix"]
    row0 = prefix if case["tails_only"] else 0
    positions = [prefix + t for t in _tails(case)]
    max_pos = _round64(max(positions) + 1 - row0)
    s.update(row0=row0, positions=positions, max_pos=max_pos, prefix_max_pos=_round64(prefix))
    s["k_prefix"] = _randn(gen, hkv, s["prefix_max_pos"], hd)
    s["v_prefix"] = _randn(gen, hkv, hd, s["prefix_max_pos"])
    s["kc"], s["vc"] = _randn(gen, b, hkv, max_pos, hd), _randn(gen, b, hkv, hd, max_pos)
    if not case["tails_only"]:
        s["kc"][:, :, :prefix] = s["k_prefix"][:, :prefix]
        s["vc"][:, :, :, :prefix] = s["v_prefix"][:, :, :prefix]
    s["qkv"] = _randn(gen, b, (hq + 2 * hkv) * hd)
    s["qkv"][:, :hq * hd] *= 1.5  # scores spread wider than unit normal: some rows weigh far more than others
    at = torch.arange(row0 + max_pos, dtype=torch.float64, device="cuda")[:, None]
    angle = at * 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    s["table"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    s["out"] = torch.zeros(b, hq * hd, dtype=torch.float16, device="cuda")
    s["pos"] = torch.tensor(positions, device="cuda")


def _prepare_logprobs(s, case, gen):
    """Logits like a trained model's: a bulk of unlikely tokens and a few likely ones in every row.  With a mask nearly
    all are -inf, and the last row has none left."""
    rows, vocab, ld = case["rows"], case["vocab"], case["vocab"] + case["pad"]
    s["logits"] = _randn(gen, rows, ld)
    s["logits"] *= 2.0
    peaks = torch.randint(vocab, (rows, 8), generator=gen, device="cuda")
    s["logits"].scatter_(1, peaks, (torch.rand(rows, 8, generator=gen, device="cuda") * 8 + 6).half())
    if case["masked"]:
        s["logits"].masked_fill_(torch.rand(rows, ld, generator=gen, device="cuda") < 0.98, -math.inf)
        s["logits"][-1] = -math.inf
    s["ids"] = torch.randint(vocab, (rows, case["n_ids"]), generator=gen, device="cuda", dtype=torch.int32)
    s["ids"][:, 0] = peaks[:, 0].int()
    s["logprob"] = torch.zeros(rows, case["n_ids"], device="cuda")
    s["entropy"] = torch.zeros(rows, device="cuda")
    s["top_ids"] = torch.zeros(rows, case["k"], dtype=torch.int32, device="cuda")
    s["top"] = torch.zeros(rows, case["k"], device="cuda")


def _prepare_fork(s, case, gen):
    layers, hkv, hd = case["layers"], case["kv_heads"], case["head_dim"]
    s["k_src"], s["v_src"] = _randn(gen, layers, hkv, case["src_max"], hd), _randn(gen, layers, hkv, hd, case["src_max"])
    s["k_dst"] = torch.full((case["dsts"], layers, hkv, case["dst_max"], hd), 1.0, dtype=torch.float16, device="cuda")
    s["v_dst"] = torch.full((case["dsts"], layers, hkv, hd, case["dst_max"]), 2.0, dtype=torch.float16, device="cuda")


def _prepare_call(s, case):
    """The library, its workspace and the arguments of the call (addresses and sizes)."""
    import __graft_entry__
    pkg = __graft_entry__.load_package()
    pkg.init(torch.cuda.current_device())
    lib = pkg.lib()
    s["check"] = pkg.capi.check
    pointers = lambda t: (ctypes.c_void_p * t.shape[0])(*[x.data_ptr() for x in t])  # noqa: E731
    if case["op"] == "shared":
        b, hq, hkv, hd = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
        # zeroed once, like the library's other workspaces, whose counters reset themselves
        s["workspace"] = torch.zeros(lib.llm_attn_shared_workspace_bytes(hq, hkv, hd, b), dtype=torch.uint8, device="cuda")
        s["call"] = lib.llm_attn_decode_rope_shared
        s["args"] = (s["qkv"].data_ptr(), s["qkv"].shape[1], s["k_prefix"].data_ptr(), s["v_prefix"].data_ptr(), case["prefix"],
                     s["prefix_max_pos"], pointers(s["kc"]), pointers(s["vc"]), (ctypes.c_int * b)(*s["positions"]), s["row0"], b,
                     s["out"].data_ptr(), hq * hd, s["table"].data_ptr(), hq, hkv, hd, s["max_pos"], s["workspace"].data_ptr())
    elif case["op"] == "logprobs":
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        s["workspace"] = torch.zeros(lib.llm_logprobs_workspace_bytes(rows, vocab, k), dtype=torch.uint8, device="cuda")
        s["call"] = lib.llm_logprobs
        s["args"] = (s["logits"].data_ptr(), s["logits"].shape[1], rows, vocab, case["temperature"], s["ids"].data_ptr(),
                     case["n_ids"], s["logprob"].data_ptr(), s["entropy"].data_ptr(), k, s["top_ids"].data_ptr() if k else None,
                     s["top"].data_ptr() if k else None, s["workspace"].data_ptr())
    else:
        s["call"] = lib.llm_kv_fork
        s["args"] = (s["k_src"].data_ptr(), s["v_src"].data_ptr(), case["src_max"], case["src_row"], pointers(s["k_dst"]),
                     pointers(s["v_dst"]), case["dsts"], case["dst_max"], case["dst_row"], case["n"], case["layers"],
                     case["kv_heads"], case["head_dim"])


def run(s):
    case = s["case"]
    if own:
        s["check"](s["call"](*s["args"], torch.cuda.current_stream().cuda_stream))
    else:
        {"shared": _plain_shared, "logprobs": _plain_logprobs, "fork": _plain_fork}[case["op"]](s, case)
    if case["op"] == "shared":
        return {"out": s["out"], "k_cache": s["kc"], "v_cache": s["vc"]}
    if case["op"] == "logprobs":
        return {"logprob": s["logprob"], "entropy": s["entropy"], "top_ids": s["top_ids"], "top": s["top"]}
    return {"k": s["k_dst"], "v": s["v_dst"]}


def _rotate(x, cs):
    """Adjacent pairs rotated by (cos, sin) pairs; fp16 results, as the library's RoPE stores them."""
    e, o = x[..., 0::2].float(), x[..., 1::2].float()
    c, sn = cs[..., 0], cs[..., 1]
    return torch.stack([c * e - sn * o, sn * e + c * o], -1).flatten(-2).half()


def _plain_shared(s, case):
    b, hq, hkv, hd, prefix = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["prefix"]
    group, row = hq // hkv, s["pos"] - s["row0"]
    cs = s["table"][s["pos"]][:, None]
    q = _rotate(s["qkv"][:, :hq * hd].view(b, hq, hd), cs).float().view(b, hkv, group, hd) / math.sqrt(hd)
    z = torch.arange(b, device="cuda")
    s["kc"][z, :, row] = _rotate(s["qkv"][:, hq * hd:(hq + hkv) * hd].view(b, hkv, hd), cs)
    s["vc"][z, :, :, row] = s["qkv"][:, (hq + hkv) * hd:].view(b, hkv, hd)
    # scores over the prefix, all sequences at once, and over each sequence's own rows
    qg = q.transpose(0, 1).reshape(hkv, b * group, hd)
    sp = torch.matmul(qg, s["k_prefix"][:, :prefix].float().transpose(1, 2).contiguous())
    sp = sp.view(hkv, b, group, prefix).transpose(0, 1)
    lo, hi = prefix - s["row0"], max(s["positions"]) - s["row0"] + 1
    st = torch.matmul(q, s["kc"][:, :, lo:hi].float().transpose(2, 3).contiguous())
    seen = torch.arange(lo, hi, device="cuda")[None] <= row[:, None]
    st = st.masked_fill(~seen[:, None, None], -math.inf)
    m = torch.maximum(sp.amax(-1, keepdim=True), st.amax(-1, keepdim=True))
    ep, et = (sp - m).exp(), (st - m).exp()
    epg = ep.transpose(0, 1).reshape(hkv, b * group, prefix)
    o = torch.matmul(epg, s["v_prefix"][:, :, :prefix].float().transpose(1, 2).contiguous()).view(hkv, b, group, hd).transpose(0, 1)
    o = o + torch.matmul(et, s["vc"][:, :, :, lo:hi].float().transpose(2, 3).contiguous())
    o = o / (ep.sum(-1, keepdim=True) + et.sum(-1, keepdim=True))
    s["out"].copy_(o.reshape(b, hq * hd))


def _plain_logprobs(s, case):
    x = s["logits"][:, :case["vocab"]].float() + 0.0  # -0 becomes +0: equal logits have equal bits
    m = x.amax(1, keepdim=True)
    y = (x - torch.where(m == -math.inf, 0.0, m)) / case["temperature"]
    e = y.exp()
    total = e.sum(1, keepdim=True)
    none = total == 0  # nothing is left of the row
    log_total = total.log()
    some = torch.where(none, 1.0, total)
    s["logprob"].copy_(torch.where(none, -math.inf, y.gather(1, s["ids"].long()) - torch.where(none, 0.0, log_total)))
    entropy = log_total - torch.where(e > 0, y * e, 0.0).sum(1, keepdim=True) / some
    s["entropy"].copy_(torch.where(none, 0.0, entropy)[:, 0])
    if case["k"]:
        top, at = x.sort(dim=1, descending=True, stable=True)
        top, at = top[:, :case["k"]], at[:, :case["k"]]
        s["top_ids"].copy_(torch.where(top == -math.inf, -1, at))
        s["top"].copy_(torch.where(top == -math.inf, -math.inf, y.gather(1, at) - torch.where(none, 0.0, log_total)))


def _plain_fork(s, case):
    a, d, n = case["src_row"], case["dst_row"], case["n"]
    s["k_dst"][:, :, :, d:d + n] = s["k_src"][:, :, a:a + n]
    s["v_dst"][..., d:d + n] = s["v_src"][..., a:a + n]


def exact(case, seed):
    """The operators from their definitions in 64 bits, sequence by sequence and in groups of rows.  Copies have no computed
    numbers; the new value rows are copies too."""
    if case["op"] == "fork":
        return None
    s = {}
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logprobs":
        _prepare_logprobs(s, case, gen)
        return _exact_logprobs(s, case)
    _prepare_shared(s, case, gen)
    hq, hkv, hd, prefix, row0 = case["heads"], case["kv_heads"], case["head_dim"], case["prefix"], s["row0"]
    out, k_cache = torch.zeros_like(s["out"], dtype=torch.float64), s["kc"].double()

    def turned(x, position):
        pairs = torch.view_as_complex(x.double().reshape(-1, hd // 2, 2).contiguous())
        angle = torch.view_as_complex(s["table"][position].double().contiguous())
        return torch.view_as_real(pairs * angle).reshape(-1, hd).half().double()

    for z, position in enumerate(s["positions"]):
        line = s["qkv"][z]
        q, k_new = turned(line[:hq * hd], position), turned(line[hq * hd:(hq + hkv) * hd], position)
        v_new = line[(hq + hkv) * hd:].double().view(hkv, hd, 1)
        k_cache[z, :, position - row0] = k_new
        for h in range(hkv):
            keys = torch.cat([s["k_prefix"][h, :prefix].double(), s["kc"][z, h, prefix - row0:position - row0].double(), k_new[h:h + 1]])
            values = torch.cat([s["v_prefix"][h, :, :prefix].double(), s["vc"][z, h, :, prefix - row0:position - row0].double(),
                                v_new[h]], 1)
            for g in range(h * hq // hkv, (h + 1) * hq // hkv):
                weights = (keys @ q[g] * hd ** -0.5).softmax(0)
                out[z, g * hd:(g + 1) * hd] = values @ weights
    return {"out": out, "k_cache": k_cache, "v_cache": None}


def _exact_logprobs(s, case):
    got = {"logprob": [], "entropy": [], "top": []}
    for at in range(0, case["rows"], 128):
        y = s["logits"][at:at + 128, :case["vocab"]].double() / case["temperature"]
        logp = y - y.logsumexp(1, keepdim=True)
        logp = torch.where(torch.isnan(logp), -math.inf, logp)  # a row without a token: every probability is zero
        got["logprob"].append(logp.gather(1, s["ids"][at:at + 128].long()))
        got["entropy"].append(-torch.where(logp == -math.inf, 0.0, logp.exp() * logp).sum(1))
        got["top"].append(logp.topk(min(case["k"], case["vocab"]), 1).values)
    return {"logprob": torch.cat(got["logprob"]), "entropy": torch.cat(got["entropy"]), "top_ids": None, "top": torch.cat(got["top"])}
