"""Arguments that the shared-prefix attention, the cache fork and the log probabilities refuse.  Every check comes before
anything touches a device, so this runs without one; the addresses are never read."""
import ctypes as C

import pytest

A = 1 << 40  # an aligned address
BIG = 1 << 36


def refused(pkg, rc, text=""):
    assert rc == pkg.capi.LLM_ERR_INVALID, rc
    msg = pkg.lib().llm_last_error().decode()
    assert text in msg, msg


def ptrs(*a):
    return (C.c_void_p * len(a))(*a)


def shared(pkg, **over):
    a = dict(qkv=A, ldq=6144, kp=A + BIG, vp=A + 2 * BIG, prefix=100, pmax=128, ks=(A + 3 * BIG, A + 4 * BIG), vs=(A + 5 * BIG, A + 6 * BIG),
             pos=(100, 150), row0=0, batch=2, out=A + 7 * BIG, ldo=4096, table=A + 8 * BIG, hq=32, hkv=8, hd=128, max_pos=256, ws=A + 9 * BIG)
    a.update(over)
    return pkg.lib().llm_attn_decode_rope_shared(
        a["qkv"], a["ldq"], a["kp"], a["vp"], a["prefix"], a["pmax"], a["ks"] and ptrs(*a["ks"]), a["vs"] and ptrs(*a["vs"]),
        a["pos"] and (C.c_int * len(a["pos"]))(*a["pos"]), a["row0"], a["batch"], a["out"], a["ldo"], a["table"], a["hq"], a["hkv"],
        a["hd"], a["max_pos"], a["ws"], None)


@pytest.mark.parametrize("over,text", [
    (dict(qkv=None), "null"), (dict(out=None), "null"), (dict(table=None), "null"), (dict(ws=None), "null"), (dict(kp=None), "null"),
    (dict(vp=None), "null"), (dict(ks=None), "null"), (dict(vs=None), "null"), (dict(pos=None), "null"),
    (dict(ks=(A, None)), "cache 1"), (dict(vs=(None, A)), "cache 0"),
    (dict(batch=0), "batch"), (dict(batch=17), "batch"), (dict(batch=-1), "batch"),
    (dict(hkv=0), "heads"), (dict(hkv=5), "heads"), (dict(hq=0), "heads"), (dict(hq=16), "not built"), (dict(hd=96), "not built"),
    (dict(hq=64, hd=64, ldq=5120), "not built"),
    (dict(max_pos=100), "multiples"), (dict(max_pos=0), "multiples"), (dict(pmax=100), "multiples"), (dict(pmax=-64), "multiples"),
    (dict(max_pos=1 << 23), "2 GiB"), (dict(pmax=1 << 23), "2 GiB"),
    (dict(prefix=129), "prefix"), (dict(prefix=-1), "prefix"), (dict(row0=-1), "row 0"), (dict(row0=101), "row 0"),
    (dict(pos=(99, 150)), "position 99"), (dict(pos=(100, 256)), "position 256"), (dict(pos=(100, -7)), "position -7"),
    (dict(pos=(100, 356), row0=100), "position 356"), (dict(pos=(100, 2 ** 31 - 1), row0=100), "position"),
    (dict(ldq=6136), "ldq"), (dict(ldq=6145), "ldq"), (dict(ldo=4095), "ldo"),
    (dict(qkv=A + 2), "aligned"), (dict(table=A + 8), "aligned"), (dict(ws=A + 4), "aligned"), (dict(kp=A + 8), "aligned"),
    (dict(ks=(A, A + 2)), "cache 1"), (dict(vs=(A + 8, A)), "cache 0"),
    (dict(ks=(A, A)), "share"), (dict(vs=(A, A)), "share"),
    (dict(ks=(A + BIG, A), vs=(A + 2 * BIG, A), row0=100, pmax=256), "the prefix lies in cache 0"), (dict(ks=(A, A + BIG)), "the prefix lies in cache 1"),
    (dict(ks=(A + BIG, A), vs=(A + 2 * BIG, A)), "whose size is another"),
])
def test_shared_attention(pkg, over, text):
    refused(pkg, shared(pkg, **over), text)


def shared_dev(pkg, **over):
    a = dict(qkv=A, ldq=6144, desc=A + BIG, po=0, co=0, mp=100, pmax=128, mt=50, batch=2, out=A, ldo=4096, table=A, hq=32, hkv=8, hd=128,
             max_pos=256, ws=A)
    a.update(over)
    return pkg.lib().llm_attn_decode_rope_shared_dev(a["qkv"], a["ldq"], a["desc"], a["po"], a["co"], a["mp"], a["pmax"], a["mt"], a["batch"],
                                                     a["out"], a["ldo"], a["table"], a["hq"], a["hkv"], a["hd"], a["max_pos"], a["ws"], None)


@pytest.mark.parametrize("over,text", [
    (dict(desc=None), "null"), (dict(qkv=None), "null"), (dict(batch=17), "batch"), (dict(hkv=3), "heads"), (dict(hd=80), "not built"),
    (dict(mp=129), "prefix"), (dict(mp=-1), "prefix"), (dict(mt=256), "rows"), (dict(mt=-1), "rows"), (dict(max_pos=65), "multiples"),
    (dict(po=4), "aligned"), (dict(co=1), "aligned"), (dict(ldo=1), "ldo"),
])
def test_shared_attention_by_descriptor(pkg, over, text):
    refused(pkg, shared_dev(pkg, **over), text)


def fork(pkg, **over):
    a = dict(k=A, v=A + BIG, smax=256, srow=0, ks=(A + 2 * BIG, A + 3 * BIG), vs=(A + 4 * BIG, A + 5 * BIG), n_dst=None, dmax=256, drow=0, n=0,
             L=32, hkv=8, hd=128)
    a.update(over)
    n_dst = len(a["ks"] or ()) if a["n_dst"] is None else a["n_dst"]
    return pkg.lib().llm_kv_fork(a["k"], a["v"], a["smax"], a["srow"], a["ks"] and ptrs(*a["ks"]), a["vs"] and ptrs(*a["vs"]), n_dst, a["dmax"],
                                 a["drow"], a["n"], a["L"], a["hkv"], a["hd"], None)


SIZE = 2 * 32 * 8 * 128 * 256  # bytes of one half of a cache above


@pytest.mark.parametrize("over,text", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(ks=None, n_dst=1), "null"), (dict(vs=None), "null"),
    (dict(ks=(None, A + 3 * BIG)), "destination 0"), (dict(vs=(A + 4 * BIG, None)), "destination 1"),
    (dict(n_dst=0), "destinations"), (dict(n_dst=17), "destinations"), (dict(n_dst=-1), "destinations"),
    (dict(L=0), "layers"), (dict(hkv=0), "layers"), (dict(L=65536, hkv=1), "layers"), (dict(hd=0), "head_dim"), (dict(hd=12), "head_dim"),
    (dict(hd=1032), "head_dim"), (dict(smax=0), "multiples"), (dict(smax=65), "multiples"), (dict(dmax=100), "multiples"), (dict(smax=(1 << 30) + 64), "2^30"), (dict(dmax=(1 << 30) + 64), "2^30"), (dict(dmax=-64), "multiples"),
    (dict(n=-1), "rows"), (dict(srow=-1), "rows"), (dict(srow=257), "rows"), (dict(srow=1, n=256), "rows"), (dict(srow=2 ** 31 - 1, n=2), "rows"),
    (dict(drow=-1), "rows"), (dict(drow=257), "rows"), (dict(drow=255, n=2), "rows"), (dict(drow=2 ** 31 - 1, n=2), "rows"),
    (dict(k=A + 2), "aligned"), (dict(v=A + 8), "aligned"), (dict(ks=(A + 2, A + 3 * BIG)), "destination 0"),
    (dict(ks=(A, A + 3 * BIG), vs=(A + BIG, A + 4 * BIG), srow=0, drow=10, n=11), "overlaps the source"),
    (dict(ks=(A, A + 3 * BIG), vs=(A + BIG, A + 4 * BIG), srow=10, drow=0, n=11), "overlaps the source"),
    (dict(ks=(A, A + 3 * BIG), vs=(A + BIG, A + 4 * BIG), srow=0, drow=100, n=11, dmax=512), "overlaps the source"),
    (dict(ks=(A + SIZE - 16, A + 3 * BIG)), "overlaps the source"), (dict(vs=(A + BIG - SIZE + 16, A + 4 * BIG)), "overlaps the source"),
    (dict(ks=(A + BIG, A + 3 * BIG)), "other half"), (dict(vs=(A, A + 4 * BIG)), "other half"),
    (dict(ks=(A + 2 * BIG, A + 2 * BIG)), "overlap"), (dict(vs=(A + 4 * BIG, A + 4 * BIG + 1024)), "overlap"), (dict(vs=(A + 2 * BIG, A + 4 * BIG)), "overlap"),
])
def test_cache_fork(pkg, over, text):
    refused(pkg, fork(pkg, **over), text)


def test_cache_fork_of_no_rows_is_a_call_that_does_nothing(pkg):
    assert fork(pkg) == pkg.capi.LLM_OK
    assert fork(pkg, srow=256, drow=256) == pkg.capi.LLM_OK
    assert fork(pkg, ks=(A,), vs=(A + BIG,), srow=3, drow=3) == pkg.capi.LLM_OK


def logprobs(pkg, **over):
    a = dict(x=A, ld=1000, rows=0, vocab=1000, t=1.0, ids=A, n=2, lp=A, ent=A, k=5, ti=A, tl=A, ws=A)
    a.update(over)
    return pkg.lib().llm_logprobs(a["x"], a["ld"], a["rows"], a["vocab"], a["t"], a["ids"], a["n"], a["lp"], a["ent"], a["k"], a["ti"], a["tl"],
                                  a["ws"], None)


@pytest.mark.parametrize("over,text", [
    (dict(x=None), "null"), (dict(ids=None), "null"), (dict(lp=None), "null"), (dict(ent=None), "null"), (dict(ti=None), "null"), (dict(tl=None), "null"),
    (dict(ws=None), "null"), (dict(rows=-1), "rows"), (dict(vocab=0), "rows"), (dict(vocab=(1 << 20) + 1, ld=1 << 21), "at most"), (dict(ld=999), "ld"), (dict(t=0.0), "temperature"),
    (dict(t=-1.0), "temperature"), (dict(t=float("nan")), "temperature"), (dict(t=float("inf")), "temperature"), (dict(t=1e-45), "temperature"),
    (dict(n=-1), "given"), (dict(n=17), "given"), (dict(k=-1), "top"), (dict(k=33), "top"), (dict(k=4, vocab=3), "top"), (dict(ws=A + 8), "aligned"),
    (dict(x=A + 1), "aligned"), (dict(ids=A + 2), "aligned"), (dict(ent=A + 1), "aligned"),
])
def test_logprobs(pkg, over, text):
    refused(pkg, logprobs(pkg, **over), text)


def test_logprobs_of_no_rows_and_of_no_tokens(pkg):
    assert logprobs(pkg) == pkg.capi.LLM_OK
    assert logprobs(pkg, n=0, ids=None, lp=None, k=0, ti=None, tl=None) == pkg.capi.LLM_OK


def test_logprobs_workspace_holds_smaller_calls_too(pkg):
    """The size never falls when rows or k grow, and is at least what a call of any smaller number of rows uses: counters for 4096
    rows, 128 bytes each, then 16 bytes and k words of 8 for each chunk of a launch's rows; a row is cut into at most 64 chunks,
    into no more than make 512 in all, rounded up to a chunk for each row."""
    need = pkg.lib().llm_logprobs_workspace_bytes

    def used(rows, k):
        return 4096 * 128 + min(rows, 4096) * min(64, -(-512 // rows)) * (16 + 8 * k)

    for vocab in (1, 64, 1000, 32003, 128256, 1 << 20):
        for k in (0, 1, 5, 32):
            last = 0
            for rows in list(range(1, 700)) + [1023, 1024, 4095, 4096, 4097, 100000]:
                size = need(rows, vocab, k)
                assert size >= last and size == need(rows, 128256, k)
                assert size >= used(rows, k) and (k == 0 or size > need(rows, vocab, k - 1))
                last = size
            assert need(600, vocab, k) >= max(used(r, k) for r in range(1, 601))


@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 512, 2 ** 31 - 4096])
def test_logprobs_of_more_rows_than_can_be_counted(pkg, rows):
    """Next to the type's end the cut of a row and the loop over slices would overflow it."""
    refused(pkg, logprobs(pkg, rows=rows, vocab=1, ld=1, k=1), "at most")


OWN = 2 * 8 * 128 * 256     # bytes of one half of an own cache of `shared` above
PREFIX = 2 * 8 * 128 * 128  # and of the prefix cache


@pytest.mark.parametrize("over,text", [
    (dict(ks=(A + 3 * BIG, A + 3 * BIG + 16)), "share"), (dict(ks=(A + 3 * BIG, A + 3 * BIG + OWN - 16)), "share"),
    (dict(vs=(A + 5 * BIG, A + 5 * BIG - OWN + 16)), "share"), (dict(vs=(A + 5 * BIG, A + 3 * BIG)), "share"),
    (dict(vs=(A + 5 * BIG, A + 4 * BIG + 256)), "halves"), (dict(ks=(A + 3 * BIG, A + 4 * BIG), vs=(A + 3 * BIG, A + 6 * BIG)), "halves"),
    (dict(kp=A + 3 * BIG + 16), "the prefix lies in cache 0"), (dict(vp=A + 6 * BIG + OWN - 16), "the prefix lies in cache 1"),
    (dict(kp=A + 6 * BIG), "the prefix lies in cache 1"), (dict(vp=A + 3 * BIG), "the prefix lies in cache 0"),
    (dict(kp=A + 4 * BIG - PREFIX + 16), "the prefix lies in cache 1"),
    (dict(kp=A + 3 * BIG + 16, vp=A + 5 * BIG + 16, pmax=256), "the prefix lies in cache 0"),
])
def test_shared_attention_on_memory_in_common(pkg, over, text):
    refused(pkg, shared(pkg, **over), text)


def test_shared_attention_takes_caches_side_by_side(pkg):
    """Caches that touch but do not overlap pass: these calls are refused for their positions, which are looked at cache by cache."""
    refused(pkg, shared(pkg, ks=(A, A + OWN), vs=(A + 2 * OWN, A + 3 * OWN), kp=A + 4 * OWN, vp=A + 4 * OWN + PREFIX, pos=(100, 256)), "position 256")
    refused(pkg, shared(pkg, ks=(A, A + OWN), vs=(A + 2 * OWN, A + 3 * OWN), kp=A, vp=A + 2 * OWN, pmax=256, pos=(100, 256)), "position 256")
